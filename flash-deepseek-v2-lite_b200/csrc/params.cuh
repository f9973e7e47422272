// Kernel parameter blocks and launcher declarations shared between the kernel
// translation units and the C-ABI layer (api.cu).
#pragma once
#include "linear.cuh"

namespace dsv2 {

// Expert-parallel peer table: every rank's peer-visible buffer as mapped in this process
// (base[rank] is local), with the same layout in every buffer:
//   xg   [world * rows_per_rank, hidden] bf16   normalised MoE inputs of all rows
//   ids  [world * rows_per_rank, 6] int32, w [...] fp32   their top-6 routing
//   part [rows_per_rank, 8, hidden] fp32         slot outputs of this rank's rows
//   ctr  two uint64 counters (128 B apart): dispatch arrivals, combine arrivals
// world == 0: single GPU (no peers).
constexpr int kMaxPeers = 8;
struct PeerTable {
  int world;
  int rank;
  char* base[kMaxPeers];
  long long xg_off, ids_off, w_off, part_off, ctr_off;
  int rows_per_rank;
  int n_moe;                  // MoE layers per step
  const long long* epoch;     // completed steps of this rank
  unsigned int wait_polls;    // poll limit of the cross-GPU waits (0 = kPeerWaitPolls)
  unsigned long long* wait_stats;  // optional [4]: dispatch waits (ns, count), combine waits (ns, count)
};

__device__ __forceinline__ unsigned long long* peer_ctr(const PeerTable& t, int rank, int which) {
  return reinterpret_cast<unsigned long long*>(t.base[rank] + t.ctr_off + which * 128);
}
// value of a counter once every rank has signalled layer `layer` of the current step
__device__ __forceinline__ unsigned long long peer_target(const PeerTable& t, int layer,
                                                          unsigned long long per_rank) {
  const unsigned long long e = static_cast<unsigned long long>(*t.epoch);
  return (e * t.n_moe + layer + 1) * static_cast<unsigned long long>(t.world) * per_rank;
}

struct RouterParams {
  const bf16* x;           // [rows, hidden] normalised activations
  long long x_row_stride;
  const void* w;           // [n_experts, hidden] gate weight, bf16 or fp32
  int w_dtype;             // 0 bf16, 2 fp32
  const float* bias;       // optional per-expert logit offset (nullptr = none)
  int rows;
  int hidden;
  int n_experts;
  float scaling;
  float* logits;           // [rows, n_experts] workspace (fp32)
  long long* topk_ids;     // [rows, 6] int64 (may be nullptr)
  int* topk_ids32;         // [rows, 6] int32 (bucketing input)
  float* topk_w;           // [rows, 6]
  // bucketing (skipped when group_offsets == nullptr)
  int expert_lo;           // first local expert
  int n_local;             // local routed experts
  int shared_lo, shared_hi;  // rows whose shared-expert routes are local
  int* group_offsets;      // [n_local + 3]
  int* route_token;        // [rows*6 + 2*(shared_hi-shared_lo)]
  int* route_slot;
  float* route_weight;
  int gather_x;            // copy each route's x row into gather_out (expert order)
  void* gather_out;
  PeerTable peers;         // world > 0: write x / ids / weights of these rows to every rank
  int row_base;            // global index of this rank's first row
  // fused residual add + RMSNorm ahead of the gate (h != nullptr; router_fused_kernel):
  // h[r] = bf16(h[r] + sum_p delta[r, p]), x_out[r] = rmsnorm(h[r]) * norm_w
  bf16* h;
  const void* delta;
  int delta_dtype;         // 0 bf16, 2 fp32 partials
  int n_delta;
  long long delta_part_stride, delta_row_stride;
  const void* norm_w;
  int norm_w_dtype;
  float eps;
  bf16* x_out;             // normalised rows (row stride x_row_stride); x == x_out then
  int* grid_sync;          // [2] grid barrier of the single-launch bucketing (nullptr: two launches)
};

struct MlaPrepParams {
  const void* qkva;            // [B, 3072 + 576]: q (16 x 192) | c_kv (512) | k_pe (64)
  int qkva_f32;                // 1: fp32 split-K partials (qkva_parts of them), 0: bf16
  int qkva_parts;
  long long qkva_part_stride;  // elements
  bf16* q_nope_out;            // optional [B, 16, 128]
  long long qkva_row_stride;
  const bf16* kv_norm_w;       // [512]
  float eps;
  const float* cos_tab;        // [positions, rope_stride] (first 32 entries used)
  const float* sin_tab;
  long long rope_stride;
  int rope_rows;
  const long long* positions;  // [1] or [B]: write position of the new token
  int pos_numel;
  bf16* cache;                 // [B, max_len, 576] (this layer)
  long long cache_b_stride;    // elements
  int max_len;
  bf16* q_pe_out;              // [B, 16, 64]
  const int* cache_rows;       // optional [B]: cache row of input row b (else b)
  int cache_batch;             // rows of the cache
  // 4-bit paged cache instead of `cache` (latent4.cuh)
  unsigned char* cache4;
  long long cache4_blocks;     // 16-token blocks of it
  const long long* slots;      // [B] slot of the new token (negative: no cache write)
};

// Rows <-> slots of the 4-bit latent cache (latent4.cu)
struct Latent4Params {
  const bf16* rows;            // write: [n, 576] source rows
  bf16* out;                   // read: [n, 576] destination rows
  long long row_stride;
  const long long* slots;      // [n], negative = padding
  long long n;
  unsigned char* cache;
  long long n_blocks;
};

// Page tables, slots and positions of a serving step (page_plan.cu)
struct PagePlanParams {
  const void* cached;          // [requests] int32 or int64 (cached64)
  int cached64;
  const int* fresh;            // [requests] tokens to append; -1 = finished
  int requests;
  int page;
  int* table;                  // [requests, width] at table_stride
  long long table_stride;
  int width;
  int* ring;                   // [ring_size] free pages
  long long ring_size;
  const long long* ring_in;    // {taken, put} counters
  long long* ring_out;
  int capacity;                // token rows
  int* token_row;
  long long* positions;
  long long* slots;
  int* cu_new;                 // [requests + 1]
  int* lens;                   // [requests]
  int* counts;                 // {tokens, pages taken, pages returned, requests not served}
  int* sync;                   // one ticket, left zero
};

// Latent attention over the paged 4-bit cache (mla_q4.cu)
struct MlaQ4Params {
  const bf16* q_abs;           // [rows, 16, 512]
  const bf16* q_pe;            // [rows, 16, 64]
  const unsigned char* cache;
  long long n_blocks;          // 16-token blocks of the cache
  const int* table;            // [seqs, width] pages at table_stride
  long long table_stride;
  int width;
  int seqs;
  int page_blocks;             // 16-token blocks per page
  const long long* positions;  // [rows], attended length = position + 1
  const int* seq_rows;         // optional [rows]: table row of each query row (negative: none)
  float scale_log2;
  bf16* o_lat;                 // [rows, 16, 512]
  int rows;
  int min_units;               // fewest units of work (16-token blocks) per CTA
  float* o_part;               // [part_slots, 16, 512] partials, two slots per CTA
  float* ml_part;              // [part_slots, 16, 2] (m in the log2 domain, l)
  int part_slots;
  int4* cuts;                  // [part_slots / 2] per CTA: {row it cuts or -1, first partial slot, number}
};

// Low-rank adapters of many requests (lora.cu)
struct LoraParams {
  const bf16* x;               // [tokens, k]
  long long x_row_stride;
  const bf16* a;               // [adapters, rank, k]
  const bf16* b;               // [adapters, n, rank]
  const int* ids;              // [tokens] (or per request with token_row), negative = none
  const int* token_row;        // optional [tokens]: request of each token (negative: none)
  const int* ranks;            // [adapters] used rank
  const float* scales;         // [adapters]
  int adapters, rank, tokens, k, n;
  int ids_len;
  float* low;                  // [low_parts, tokens, rank] work buffer (long runs: the first part, in adapter order)
  int low_parts;               // k splits of the first product
  int* order;                  // [3, tokens] work buffer: tokens by adapter, adapters, ranks (nullptr: as they come)
  const float* base;           // optional fp32 partials of the shared projection, summed in order
  int base_parts;
  long long base_part_stride, base_row_stride;
  void* y;                     // [tokens, n] bf16 or fp32
  int y_f32;
  long long y_row_stride;
  const bf16* w;               // few tokens: the shared projection's weights, [n, k] (else null)
  long long w_row_stride;
  bf16* xs;                    // long runs of tokens: [tokens, k] work buffer, x in adapter order
  int* lists;                  // [ceil(tokens / 256), 2 + 512 ceil(rank / 16)] work buffer, adapters of each token tile
};

struct MlaDecodeParams {
  const bf16* q_abs;           // [B, 16, 512]
  const bf16* q_pe;            // [B, 16, 64]
  const bf16* cache;           // [B, max_len, 576]
  long long cache_b_stride;
  int max_len;
  const long long* positions;  // [1] or [B]; attended length = position + 1
  int pos_numel;
  float scale_log2;            // softmax_scale * log2(e)
  // mma.sync kernel: split_len = fewest positions per CTA, o_part / ml_part hold
  // batch * n_splits partial slots (two per CTA), row_sync = per-row merge tickets.
  // tcgen05 kernel: split_len = positions per split, o_part [B, n_splits, 16, 512].
  int split_len;
  int n_splits;
  float* o_part;
  float* ml_part;              // (m in log2 domain, l) per head and partial
  bf16* o_lat;                 // [B, 16, 512] output
  int inputs_prior;            // q_pe / positions / cache written >= 2 launches earlier
  int* row_sync;               // [B] zero-initialised, left zero
  int batch;
  const int* cache_rows;       // optional [B]: cache row read by query row b (else b)
  int cache_batch;             // rows of the cache
  int* part_count;             // optional (B = 1): partials left unmerged; [first CTA, count]
};

// norm.cu
cudaError_t launch_rmsnorm(const void*, long long, int, const void*, int, void*, long long, int, int,
                           float, cudaStream_t);
cudaError_t launch_add_rmsnorm(void*, void*, const void*, int, int, long long, long long,
                               const void*, int, void*, int, int, float, cudaStream_t,
                               const PeerTable* peers = nullptr, int layer = 0);
cudaError_t launch_embed_rmsnorm(const long long*, const void*, long long, const void*, int, void*,
                                 void*, int, int, float, cudaStream_t);
cudaError_t launch_residual_add(const void*, const void*, void*, long long, int, cudaStream_t);
cudaError_t launch_silu_mul(const void*, const void*, void*, long long, cudaStream_t);
cudaError_t launch_sum_partials(const float* part, int n_parts, long long ps, long long rs, void* out,
                               int out_f32, long long ors, int rows, int cols, cudaStream_t st);
cudaError_t launch_prepare_decode_inputs(const long long*, int, long long*, long long, long long*,
                                         long long, const long long*, int, int, cudaStream_t);
cudaError_t launch_copy_token_to_cache(const void*, const long long*, void*, const long long*,
                                       const long long*, int, int, int, int, int, int,
                                       cudaStream_t);
cudaError_t launch_advance_positions(long long*, int, cudaStream_t);
cudaError_t launch_argmax_finalize(const unsigned long long* keys, int n_blocks, long long key_stride,
                                   int n_tokens, long long* next_ids, long long* input_ids,
                                   long long* positions, int pos_numel, long long* step_counter,
                                   const long long* served, int* missed, cudaStream_t st);
// router.cu
cudaError_t launch_router(const RouterParams&, int max_clusters, int num_sms, cudaStream_t);
cudaError_t router_fused_max_clusters(int* n);
cudaError_t launch_bucket(const int*, const float*, int, int, int, int, int, int*, int*, int*,
                          float*, const void*, long long, void*, int, int, cudaStream_t,
                          const PeerTable* peers, int layer);
cudaError_t launch_softmax_topk(const float*, int, int, float, long long*, int*, float*,
                                cudaStream_t);
cudaError_t launch_gather_rows(const void*, long long, const int*, const int*, int, void*, int,
                               int, cudaStream_t);
// mla.cu
cudaError_t launch_mla_prep(const MlaPrepParams&, int, cudaStream_t);
cudaError_t launch_mla_prep_q4(const MlaPrepParams&, int, cudaStream_t);
// latent4.cu, page_plan.cu, mla_q4.cu, lora.cu
cudaError_t launch_latent4_write(const Latent4Params&, cudaStream_t);
cudaError_t launch_latent4_read(const Latent4Params&, cudaStream_t);
cudaError_t launch_page_plan(const PagePlanParams&, int num_sms, cudaStream_t);
cudaError_t mla_q4_init();
cudaError_t launch_mla_q4(const MlaQ4Params&, int num_sms, cudaStream_t);
cudaError_t launch_lora(const LoraParams&, int num_sms, cudaStream_t);
cudaError_t launch_lora_rows(const LoraParams&, int num_sms, cudaStream_t);
cudaError_t lora_gemm_init();
int lora_gemm_tile(int tokens, int n, int num_sms);
cudaError_t launch_lora_gemm(const LoraParams&, const CUtensorMap& tm_x, const CUtensorMap& tm_w, int n_tile, int num_sms,
                             cudaStream_t);
cudaError_t mla_decode_init();
int mla_decode_grid(const MlaDecodeParams&, int num_sms, long long part_slots);
cudaError_t launch_mla_decode(const MlaDecodeParams&, const CUtensorMap& tm_kv, const CUtensorMap& tm_qa,
                              const CUtensorMap& tm_qp, int grid, cudaStream_t);
cudaError_t launch_mla_combine(const MlaDecodeParams&, int, cudaStream_t);
// linear_tc.cu (TcShape, tc_launch_shape and launch_linear_tc_impl are defined there; the
// unity build includes it before api.cu)
cudaError_t linear_tc_init();

}  // namespace dsv2

// Low-rank adapters of many requests beside a shared projection:
//   low[t, j] = scale_a * sum_k x[t, k] A_a[j, k]           (fp32, j < rank of a)
//   y[t, n]   = sum of the shared projection's partials + sum_j low[t, j] B_a[n, j]
// with a = the adapter of token t (none: y is the shared projection alone).
//
// Tokens are ordered by adapter (lora_sort_kernel; up to 16 tokens need no order) and taken 16 at a
// time, the M of an mma.sync.  A tile runs once for every adapter that it holds, with that adapter's
// rows stored, so its weights are read once per 16 tokens instead of once per token; the two
// products together have 2 rank (k + n) operations a token against the shared projection's 2 k n,
// and are bound by reading A, B, x and the partials.  Fragments come straight from global memory,
// 16 bytes a lane: which k the lanes of a quad hold is free as long as both operands agree, so
// lane tq of a quad takes 8 consecutive k of every 32.
//
// With the shared projection (2048 -> 3648): 1 token 7.3 us, 15 MB and two launches (lora_few_kernel); 200
// tokens of 40 adapters of rank 64 29.6 us, 43 MB, of which the projection takes about 9 and the rest is
// latency of the order, first and second product.  Long runs of tokens: lora_gemm.cu.
#include "params.cuh"

namespace dsv2 {

constexpr int kLoraTile = 16;      // tokens of a tile
constexpr int kLoraLowWarps = 4;   // warps of the first product, each a quarter of the CTA's k range
constexpr int kLoraOutWarps = 8;   // warps of the second product
constexpr int kLoraOutCols = 256;  // columns of one of its CTAs, 32 a warp

// adapter of token t, -1 = none (an id that names no adapter also raises the error word)
__device__ __forceinline__ int lora_id(const LoraParams& p, int t) {
  int r = t;
  if (p.token_row) r = p.token_row[t];
  if (r < 0) return -1;
  if (r >= p.ids_len) {
    set_device_error(kErrIndex);
    return -1;
  }
  const int a = p.ids[r];
  if (a >= p.adapters) {
    set_device_error(kErrIndex);
    return -1;
  }
  return a < 0 ? -1 : a;
}

// order[pos] = t, order[tokens + pos] = its adapter and order[2 tokens + pos] the adapter's rank, with pos = #{u: id_u < id_t} + #{u < t: id_u =
// id_t}: every pair of tokens is compared once (16 million at 4096 tokens), with no histogram over
// the adapters, whose number is the caller's.  A CTA's warps share 32 tokens: lane = token, warp = a part of
// the others.
constexpr int kLoraSortChunk = 4096;
constexpr int kLoraSortThreads = 1024;
__global__ __launch_bounds__(kLoraSortThreads) void lora_sort_kernel(const LoraParams p) {
  pdl_enter();
  __shared__ __align__(16) int s_id[kLoraSortChunk];
  __shared__ int s_before[kLoraSortThreads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 32 + lane;
  const int mine = t < p.tokens ? lora_id(p, t) : 0;
  int before = 0;
  for (int u0 = 0; u0 < p.tokens; u0 += kLoraSortChunk) {
    __syncthreads();
    int v[kLoraSortChunk / kLoraSortThreads];
#pragma unroll
    for (int i = 0; i < kLoraSortChunk / kLoraSortThreads; ++i) {
      const int u = u0 + i * kLoraSortThreads + threadIdx.x;
      v[i] = u < p.tokens ? lora_id(p, u) : 0x7fffffff;
    }
#pragma unroll
    for (int i = 0; i < kLoraSortChunk / kLoraSortThreads; ++i) s_id[i * kLoraSortThreads + threadIdx.x] = v[i];
    __syncthreads();
    const int n = min(kLoraSortChunk, p.tokens - u0);
    const int4* q = reinterpret_cast<const int4*>(s_id);
    const int rel = t - u0;
    // w < mine, or equal and earlier: an equal one counts when its index is below this token's.  The
    // CTA's tokens are 32 in a row, so only the quads among them need a look at each index
    const int r0 = rel - lane;
#pragma unroll 4
    for (int i = warp; i < (n + 3) / 4; i += kLoraSortThreads / 32) {
      const int4 w = q[i];
      if (4 * i >= r0 && 4 * i < r0 + 32) {
        before += (w.x < mine + (4 * i < rel)) + (w.y < mine + (4 * i + 1 < rel)) + (w.z < mine + (4 * i + 2 < rel)) +
                  (w.w < mine + (4 * i + 3 < rel));
      } else {
        const int m = mine + (4 * i < r0);
        before += (w.x < m) + (w.y < m) + (w.z < m) + (w.w < m);
      }
    }
  }
  s_before[threadIdx.x] = before;
  __syncthreads();
  if (warp == 0 && t < p.tokens) {
    for (int w = 1; w < kLoraSortThreads / 32; ++w) before += s_before[w * 32 + lane];
    p.order[before] = t;
    p.order[p.tokens + before] = mine;
    p.order[2 * p.tokens + before] = mine >= 0 ? min(max(p.ranks[mine], 0), p.rank) : 0;
  }
}

// The 16 tokens of a tile and its adapters, in shared memory.
struct LoraTile {
  int tok[kLoraTile];    // token of each row, -1 = none
  int which[kLoraTile];  // the row's adapter as an index into list, -1 = a token without one, -2 = no token
  int list[kLoraTile];   // the different adapters, their ranks
  int rank[kLoraTile];
  int n;
};
__device__ __forceinline__ void lora_tile(const LoraParams& p, int tile, LoraTile& s) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, i = tile * kLoraTile + lane;
    const bool in = lane < kLoraTile && i < p.tokens;
    const int t = in ? (p.order ? p.order[i] : i) : -1;
    const int a = in ? (p.order ? p.order[p.tokens + i] : lora_id(p, i)) : -2;
    const int rank = a < 0 ? 0 : p.order ? p.order[2 * p.tokens + i] : min(max(p.ranks[a], 0), p.rank);
    const unsigned same = __match_any_sync(0xffffffffu, a);
    const int leader = __ffs(same) - 1;
    const unsigned leaders = __ballot_sync(0xffffffffu, a >= 0 && leader == lane);
    const int idx = __popc(leaders & ((1u << leader) - 1));
    if (lane < kLoraTile) {
      s.tok[lane] = t;
      s.which[lane] = a >= 0 ? idx : a;
      if (a >= 0 && leader == lane) {
        s.list[idx] = a;
        s.rank[idx] = rank;
      }
    }
    if (lane == 0) s.n = __popc(leaders);
  }
  __syncthreads();
}

__device__ __forceinline__ uint4 ld_or_zero(const void* q, bool in) {
  return in ? __ldg(reinterpret_cast<const uint4*>(q)) : make_uint4(0, 0, 0, 0);
}

// Tiles of the GEMM of lora_gemm.cu.
constexpr int kLgRows = 128;          // tokens of a CTA's half of a tile
constexpr int kLgM = 2 * kLgRows;     // tokens of a tile
constexpr int kLgPiece = 16;          // ranks of a piece, the k of one tcgen05.mma
// ints of a tile's list: the number of pieces, one unused, then (adapter, first rank | ranks << 16) each
__host__ __device__ constexpr long long lg_list_ints(int rank) {
  return 2 + 2LL * kLgM * ((rank + kLgPiece - 1) / kLgPiece);
}
// The pieces of a tile, by one warp.
__device__ __forceinline__ void lora_list_pieces(const LoraParams& p, int tile) {
  const int lane = threadIdx.x & 31;
  int* list = p.lists + tile * lg_list_ints(p.rank);
  int ad[kLgM / 32], before[kLgM / 32], ranks[kLgM / 32];   // all loads under way together
#pragma unroll
  for (int q = 0; q < kLgM / 32; ++q) {
    const int pos = tile * kLgM + q * 32 + lane;
    ad[q] = pos < p.tokens ? p.order[p.tokens + pos] : -1;
    before[q] = pos < p.tokens && q * 32 + lane > 0 ? p.order[p.tokens + pos - 1] : -1;
    ranks[q] = pos < p.tokens ? p.order[2 * p.tokens + pos] : 0;
  }
  int n = 0;
#pragma unroll
  for (int q = 0; q < kLgM / 32; ++q) {
    // tokens are in adapter order: the first of each adapter lists its pieces
    const int a = ad[q], rank = a >= 0 && a != before[q] ? ranks[q] : 0, mine = (rank + kLgPiece - 1) / kLgPiece;
    int at = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, at, d);
      if (lane >= d) at += u;
    }
    const int sum = __shfl_sync(0xffffffffu, at, 31);
    at += n - mine;
    for (int c = 0; c < mine; ++c) {
      list[2 + 2 * (at + c)] = a;
      list[2 + 2 * (at + c) + 1] = c * kLgPiece | min(rank - c * kLgPiece, kLgPiece) << 16;
    }
    n += sum;
  }
  if (lane == 0) list[0] = n;
}

// bf16 values that are not finite -> 0
__device__ __forceinline__ bool drop_nonfinite(uint4& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
  __nv_bfloat162 sick = zero;   // 0 * x + 0 is a NaN for those alone
#pragma unroll
  for (int i = 0; i < 4; ++i) sick = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(w + i), zero, sick);
  if (!(__hisnan(__low2bfloat16(sick)) || __hisnan(__high2bfloat16(sick)))) return false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
  }
  return true;
}

__device__ __forceinline__ float ld_cluster_f32(const float* local, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(local, rank)) : "memory");
  return v;
}

// low partials of one tile and k split: low[split, t, j].  NT = rank / 8 n-tiles of 8 ranks.  For the
// GEMM of lora_gemm.cu (kSorted) the tile's rows of xs and the whole low, both in adapter order, and the
// pieces of each tile of that GEMM: one pass over x where a low of its own and a gather take two
// (4001 tokens, k 2048, rank 32: 16 us for both, 16 + 10 us apart).  (Two CTAs an SM: at rank 64 the compiler
// otherwise keeps fewer loads under way, 3800 tokens 53 us against 31.)  The k splits are then the CTAs of
// a cluster, which sum through each other's shared memory.
template <int NT, int kWarps, bool kSorted>
__global__ __launch_bounds__(kWarps * 32, kSorted && NT == 8 ? 2 : 0) void lora_low_kernel(const LoraParams p) {
  pdl_enter();
  __shared__ LoraTile s;
  __shared__ float s_sum[kWarps][kLoraTile][8 * NT + 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  lora_tile(p, blockIdx.x, s);
  if (kSorted) {
    if (blockIdx.x % (kLgM / kLoraTile) == 0 && blockIdx.y == 0 && warp == kWarps - 1) lora_list_pieces(p, blockIdx.x / (kLgM / kLoraTile));
    for (int r = blockIdx.y * kWarps + warp; r < kLoraTile && s.tok[r] >= 0; r += gridDim.y * kWarps) {
      const uint4* src = reinterpret_cast<const uint4*>(p.x + s.tok[r] * p.x_row_stride);
      uint4* dst = reinterpret_cast<uint4*>(p.xs + (blockIdx.x * kLoraTile + r) * static_cast<long long>(p.k));
#pragma unroll 8
      for (int j = lane; j < p.k / 8; j += 32) dst[j] = __ldg(src + j);
    }
  }
  // this CTA's k range, in steps of 32, and this warp's part of it
  const int steps = (p.k + 31) / 32, splits = gridDim.y * kWarps, part = blockIdx.y * kWarps + warp;
  const int k0 = static_cast<int>(static_cast<long long>(steps) * part / splits) * 32;
  const int k1 = static_cast<int>(static_cast<long long>(steps) * (part + 1) / splits) * 32;
  const int t0 = s.tok[gq], t1 = s.tok[gq + 8];
  const bf16* x0 = p.x + (t0 >= 0 ? t0 : 0) * p.x_row_stride;
  const bf16* x1 = p.x + (t1 >= 0 ? t1 : 0) * p.x_row_stride;
  auto sync = [&]() {   // of those that share the sums
    if (kSorted && gridDim.y > 1) {
      cluster_arrive_release();
      cluster_wait_acquire();
    } else {
      __syncthreads();
    }
  };
  // the adapters of a tile are dealt out to the CTAs that share it
  for (int ai = blockIdx.z; ai < s.n; ai += gridDim.z) {
    const int a = s.list[ai], rank = s.rank[ai], nt = (rank + 7) / 8;
    const bf16* w = p.a + static_cast<long long>(a) * p.rank * p.k;
    const float scale = p.scales[a];
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const bool m0 = s.which[gq] == ai, m1 = s.which[gq + 8] == ai;
#pragma unroll (NT <= 4 ? 4 : 2)
    for (int k = k0 + 8 * tq; k < k1; k += 32) {
      const bool in = k < p.k;
      const uint4 u0 = ld_or_zero(x0 + k, in && m0), u1 = ld_or_zero(x1 + k, in && m1);
      uint4 b[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) b[n] = ld_or_zero(w + (8 * n + gq) * static_cast<long long>(p.k) + k, in && n < nt);
      const uint32_t f0[4] = {u0.x, u1.x, u0.y, u1.y}, f1[4] = {u0.z, u1.z, u0.w, u1.w};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n < nt) {
          mma_bf16_16816(acc[n], f0, b[n].x, b[n].y);
          mma_bf16_16816(acc[n], f1, b[n].z, b[n].w);
        }
      }
    }
    sync();   // the previous adapter's sums have been read
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s_sum[warp][gq][8 * n + 2 * tq] = acc[n][0];
      s_sum[warp][gq][8 * n + 2 * tq + 1] = acc[n][1];
      s_sum[warp][gq + 8][8 * n + 2 * tq] = acc[n][2];
      s_sum[warp][gq + 8][8 * n + 2 * tq + 1] = acc[n][3];
    }
    sync();
    const int part0 = kSorted ? blockIdx.y * kWarps * 32 : 0, parts = kSorted ? gridDim.y * kWarps * 32 : kWarps * 32;
    for (int i = part0 + threadIdx.x; i < kLoraTile * 8 * NT; i += parts) {
      const int r = i / (8 * NT), j = i % (8 * NT);
      if (s.which[r] != ai || j >= p.rank) continue;
      float v = 0.f;
      if (kSorted && gridDim.y > 1) {
        for (uint32_t c = 0; c < gridDim.y; ++c) {
#pragma unroll
          for (int q = 0; q < kWarps; ++q) v += ld_cluster_f32(&s_sum[q][r][j], c);
        }
      } else {
#pragma unroll
        for (int q = 0; q < kWarps; ++q) v += s_sum[q][r][j];
      }
      // columns past the adapter's rank hold whatever its padding holds
      v = j < rank ? v * scale : 0.f;
      const long long row = kSorted ? blockIdx.x * kLoraTile + r : static_cast<long long>(blockIdx.y) * p.tokens + s.tok[r];
      p.low[row * p.rank + j] = v;
    }
  }
  if (kSorted && gridDim.y > 1) sync();   // nobody reads this CTA's sums any more
}

// y: a tile of 16 tokens x kChunks blocks of 256 columns.  A warp takes 32 columns as two pairs of
// n-tiles; column 2 q + e of n-tile u of a pair is column 4 q + 2 u + e of its 16, so that a lane ends
// with 4 consecutive columns: whole sectors of the partials in, of y out.  low is used as the sum of
// two bf16 numbers (16 significant bits), so that it adds no rounding of its own to y.  A CTA writes
// the rows of its adapters (blockIdx.z 0 also those of none).
template <int kChunks>
__global__ __launch_bounds__(kLoraOutWarps * 32, 3) void lora_out_kernel(const LoraParams p) {
  pdl_enter();
  __shared__ LoraTile s;
  __shared__ __align__(16) uint32_t s_hi[kLoraTile][68], s_lo[kLoraTile][68];   // bf16 pairs, up to 128 ranks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  lora_tile(p, blockIdx.y, s);
  const int z = blockIdx.z, zs = gridDim.z;   // zs is a power of two
  if (z > 0 && z >= s.n) return;
  const int ad0 = s.which[gq], ad1 = s.which[gq + 8];
  // this CTA's rows
  const bool own0 = ad0 >= 0 ? (ad0 & (zs - 1)) == z : ad0 == -1 && z == 0;
  const bool own1 = ad1 >= 0 ? (ad1 & (zs - 1)) == z : ad1 == -1 && z == 0;
  // the tile's low rows: the k splits summed in order, as high and low bf16 parts; 0 past the rank
  const int shift = p.rank <= 32 ? 4 : p.rank <= 64 ? 5 : 6;   // log2 of the pairs staged per row
  for (int i = threadIdx.x; i < kLoraTile << shift; i += kLoraOutWarps * 32) {
    const int r = i >> shift, pair = i & ((1 << shift) - 1), j = 2 * pair;
    float v0 = 0.f, v1 = 0.f;
    if (s.which[r] >= 0 && j < p.rank) {
      const float* src = p.low + static_cast<long long>(s.tok[r]) * p.rank + j;
      const long long step = static_cast<long long>(p.tokens) * p.rank;
#pragma unroll 4
      for (int q = 0; q < p.low_parts; ++q, src += step) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
        v0 += v.x;
        v1 += v.y;
      }
    }
    const uint32_t hi = pack_bf16x2(v0, v1);
    s_hi[r][pair] = hi;
    // (an infinite high part is all there is: inf - inf would make it a NaN)
    s_lo[r][pair] = pack_bf16x2(isinf(bf16lo(hi)) ? 0.f : v0 - bf16lo(hi), isinf(bf16hi(hi)) ? 0.f : v1 - bf16hi(hi));
  }
  __syncthreads();
  const int col = blockIdx.x * (kChunks * kLoraOutCols) + warp * 32;
  const float* base0 = p.base + (own0 ? s.tok[gq] * p.base_row_stride : 0) + col + 4 * tq;
  const float* base1 = p.base + (own1 ? s.tok[gq + 8] * p.base_row_stride : 0) + col + 4 * tq;
  const long long y0 = (own0 ? s.tok[gq] * p.y_row_stride : 0) + col + 4 * tq;
  const long long y1 = (own1 ? s.tok[gq + 8] * p.y_row_stride : 0) + col + 4 * tq;
#pragma unroll
  for (int ch = 0; ch < kChunks; ++ch) {
    const int n0 = col + ch * kLoraOutCols;
    if (n0 >= p.n) break;
    // shared projection: 4 consecutive columns of two tokens per pair of n-tiles
    float4 v[2][2];   // [pair][token]
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h][0] = v[h][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool in0 = n0 + 4 * tq < p.n, in1 = n0 + 16 + 4 * tq < p.n;
    const float *q0 = base0 + ch * kLoraOutCols, *q1 = base1 + ch * kLoraOutCols;
    for (int q = 0; q < p.base_parts; ++q, q0 += p.base_part_stride, q1 += p.base_part_stride) {
      const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 x00 = own0 && in0 ? __ldcg(reinterpret_cast<const float4*>(q0)) : zero;
      const float4 x10 = own0 && in1 ? __ldcg(reinterpret_cast<const float4*>(q0 + 16)) : zero;
      const float4 x01 = own1 && in0 ? __ldcg(reinterpret_cast<const float4*>(q1)) : zero;
      const float4 x11 = own1 && in1 ? __ldcg(reinterpret_cast<const float4*>(q1 + 16)) : zero;
      v[0][0] = make_float4(v[0][0].x + x00.x, v[0][0].y + x00.y, v[0][0].z + x00.z, v[0][0].w + x00.w);
      v[1][0] = make_float4(v[1][0].x + x10.x, v[1][0].y + x10.y, v[1][0].z + x10.z, v[1][0].w + x10.w);
      v[0][1] = make_float4(v[0][1].x + x01.x, v[0][1].y + x01.y, v[0][1].z + x01.z, v[0][1].w + x01.w);
      v[1][1] = make_float4(v[1][1].x + x11.x, v[1][1].y + x11.y, v[1][1].z + x11.z, v[1][1].w + x11.w);
    }
    float acc[4][4];   // n-tiles 0, 1: columns n0 .. + 16; 2, 3: + 16 .. + 32
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      acc[2 * h][0] = v[h][0].x;
      acc[2 * h][1] = v[h][0].y;
      acc[2 * h + 1][0] = v[h][0].z;
      acc[2 * h + 1][1] = v[h][0].w;
      acc[2 * h][2] = v[h][1].x;
      acc[2 * h][3] = v[h][1].y;
      acc[2 * h + 1][2] = v[h][1].z;
      acc[2 * h + 1][3] = v[h][1].w;
    }
    const int nb = n0 + 4 * (gq >> 1) + (gq & 1);   // row of B of column gq of n-tile 0; + 2, + 16, + 18
    for (int ai = z; ai < s.n; ai += zs) {
      const int rank = s.rank[ai];
      const bf16* src = p.b + (static_cast<long long>(s.list[ai]) * p.n + nb) * p.rank + 8 * tq;
      for (int j = 0; j < rank; j += 32, src += 32) {
        // lane tq takes ranks j + 8 tq .. + 8 of four rows of B
        const int have = rank - j - 8 * tq;   // ranks of this lane's 8 that exist
        uint4 b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int dn = 16 * (u >> 1) + 2 * (u & 1);
          b[u] = ld_or_zero(src + dn * p.rank, have > 0 && nb + dn < p.n);
        }
        if (have > 0 && have < 8) {
          // padding past the rank may be anything, and 0 * NaN is not 0
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t* bw = reinterpret_cast<uint32_t*>(&b[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (2 * i >= have) bw[i] = 0;
              else if (2 * i + 1 >= have) bw[i] &= 0xffffu;
            }
          }
        }
        const int jw = j / 2 + 4 * tq;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 h0 = ad0 == ai ? *reinterpret_cast<const uint4*>(&s_hi[gq][jw]) : zero;
        const uint4 h1 = ad1 == ai ? *reinterpret_cast<const uint4*>(&s_hi[gq + 8][jw]) : zero;
        const uint4 l0 = ad0 == ai ? *reinterpret_cast<const uint4*>(&s_lo[gq][jw]) : zero;
        const uint4 l1 = ad1 == ai ? *reinterpret_cast<const uint4*>(&s_lo[gq + 8][jw]) : zero;
        const uint32_t ah0[4] = {h0.x, h1.x, h0.y, h1.y}, ah1[4] = {h0.z, h1.z, h0.w, h1.w};
        const uint32_t al0[4] = {l0.x, l1.x, l0.y, l1.y}, al1[4] = {l0.z, l1.z, l0.w, l1.w};
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float d[4] = {acc[u][0], acc[u][1], acc[u][2], acc[u][3]};
          mma_bf16_16816(d, ah0, b[u].x, b[u].y);
          mma_bf16_16816(d, ah1, b[u].z, b[u].w);
          drop_nonfinite(b[u]);   // the low part may have the other sign or be 0: infinities are the high part's
          __syncwarp();
          mma_bf16_16816(d, al0, b[u].x, b[u].y);
          mma_bf16_16816(d, al1, b[u].z, b[u].w);
          // other adapters' rows have zeros here, but 0 times an infinity of this B would still reach them
          if (ad0 == ai) acc[u][0] = d[0], acc[u][1] = d[1];
          if (ad1 == ai) acc[u][2] = d[2], acc[u][3] = d[3];
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!(h ? in1 : in0)) continue;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (!(c ? own1 : own0)) continue;
        const float v0 = acc[2 * h][2 * c], v1 = acc[2 * h][2 * c + 1], v2 = acc[2 * h + 1][2 * c], v3 = acc[2 * h + 1][2 * c + 1];
        const long long off = (c ? y1 : y0) + ch * kLoraOutCols + 16 * h;
        if (p.y_f32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.y) + off) = make_float4(v0, v1, v2, v3);
        else *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(p.y) + off) = make_uint2(pack_bf16x2(v0, v1), pack_bf16x2(v2, v3));
      }
    }
  }
}

// Few tokens (kGroups x 8): the shared projection and the second product in one launch, 16 columns of y
// a CTA.  Eight warps take a part of k each, W as the mma's 16 rows and tokens as its 8 columns; the first
// 256 of each part of W are requested before the wait for the first product's launch.  Then a thread adds
// the ranks (with 8 tokens: half of them) of one of the 16 x tokens results.  Bound by reading W (15 MB)
// and the chain of two launches: 1 token of rank 16, 2048 -> 3648, 7.3 us (2.1 TB/s); 8 of rank 32 9.4; as
// projection, first and second product 9.2 and 12.8.
constexpr int kLoraFewCols = 16, kLoraFewWarps = 8, kLoraFewAhead = 8;
template <int kGroups>
__global__ __launch_bounds__(kLoraFewWarps * 32, 2) void lora_few_kernel(const LoraParams p) {
  constexpr int kTok = 8 * kGroups, kHalves = kGroups == 1 ? 2 : 1;
  __shared__ float s_red[kLoraFewWarps][kTok][kLoraFewCols + 1];
  __shared__ float s_low[kTok][128];
  __shared__ float s_half[8][kLoraFewCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int n0 = blockIdx.x * kLoraFewCols;
  const int steps = (p.k + 31) / 32;
  const int k0 = steps * warp / kLoraFewWarps * 32, k1 = steps * (warp + 1) / kLoraFewWarps * 32;
  const bool in0 = n0 + gq < p.n, in1 = n0 + gq + 8 < p.n;
  const bf16* w0 = p.w + (in0 ? n0 + gq : 0) * p.w_row_stride;
  const bf16* w1 = p.w + (in1 ? n0 + gq + 8 : 0) * p.w_row_stride;
  uint4 a0[kLoraFewAhead], a1[kLoraFewAhead];
  auto load_w = [&](int k) {
#pragma unroll
    for (int i = 0; i < kLoraFewAhead; ++i) {
      const int kk = k + 32 * i + 8 * tq;
      const bool in = kk < k1 && kk < p.k;
      a0[i] = ld_or_zero(w0 + kk, in && in0);
      a1[i] = ld_or_zero(w1 + kk, in && in1);
    }
  };
  load_w(k0);
  pdl_enter();
  // low of the tokens, its pieces summed in order
  for (int i = threadIdx.x; i < p.tokens * p.rank; i += kLoraFewWarps * 32) {
    const int t = i / p.rank;
    float v = 0.f;
    if (lora_id(p, t) >= 0) {
#pragma unroll 8
      for (int q = 0; q < p.low_parts; ++q) v += __ldcg(p.low + static_cast<long long>(q) * p.tokens * p.rank + i);
    }
    s_low[t][i % p.rank] = v;
  }
  float acc[kGroups][4];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.f;
  for (int k = k0; k < k1; k += 32 * kLoraFewAhead) {
    if (k > k0) load_w(k);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int t = 8 * g + gq;
      const bf16* x = p.x + (t < p.tokens ? t : 0) * p.x_row_stride;
      uint4 u[kLoraFewAhead];
#pragma unroll
      for (int i = 0; i < kLoraFewAhead; ++i) {
        const int kk = k + 32 * i + 8 * tq;
        u[i] = ld_or_zero(x + kk, kk < k1 && kk < p.k && t < p.tokens);
      }
#pragma unroll
      for (int i = 0; i < kLoraFewAhead; ++i) {
        const uint32_t f0[4] = {a0[i].x, a1[i].x, a0[i].y, a1[i].y}, f1[4] = {a0[i].z, a1[i].z, a0[i].w, a1[i].w};
        mma_bf16_16816(acc[g], f0, u[i].x, u[i].y);
        mma_bf16_16816(acc[g], f1, u[i].z, u[i].w);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    s_red[warp][8 * g + 2 * tq][gq] = acc[g][0];
    s_red[warp][8 * g + 2 * tq + 1][gq] = acc[g][1];
    s_red[warp][8 * g + 2 * tq][gq + 8] = acc[g][2];
    s_red[warp][8 * g + 2 * tq + 1][gq + 8] = acc[g][3];
  }
  __syncthreads();
#pragma unroll
  for (int o = threadIdx.x; o < kLoraFewCols * kTok * kHalves; o += kLoraFewWarps * 32) {
    const int col = o % kLoraFewCols, t = o / kLoraFewCols % kTok;
    const bool upper = o >= kLoraFewCols * kTok, mine = t < p.tokens && n0 + col < p.n;
    const int id = mine ? lora_id(p, t) : -1;
    const int rank = id >= 0 ? min(max(p.ranks[id], 0), p.rank) : 0;
    const int mid = kHalves == 2 ? p.rank / 16 * 8 : p.rank, j0 = upper ? mid : 0, j1 = min(upper ? p.rank : mid, rank);
    const bf16* b = p.b + (static_cast<long long>(max(id, 0)) * p.n + (mine ? n0 + col : 0)) * p.rank;
    float v = 0.f;
#pragma unroll 4
    for (int j = j0; j < j1; j += 8) {
      const uint4 c = __ldg(reinterpret_cast<const uint4*>(b + j));
      const uint32_t wd[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // what lies past the rank may be anything
        if (j + 2 * i < j1) v += s_low[t][j + 2 * i] * bf16lo(wd[i]);
        if (j + 2 * i + 1 < j1) v += s_low[t][j + 2 * i + 1] * bf16hi(wd[i]);
      }
    }
    if (kHalves == 2) {   // one round, of all threads
      if (upper) s_half[t][col] = v;
      __syncthreads();
      if (!upper) v += s_half[t][col];
    }
    if (upper || !mine) continue;
    float base = 0.f;
#pragma unroll
    for (int q = 0; q < kLoraFewWarps; ++q) base += s_red[q][t][col];
    v += base;
    const long long at = t * p.y_row_stride + n0 + col;
    if (p.y_f32) reinterpret_cast<float*>(p.y)[at] = v;
    else reinterpret_cast<bf16*>(p.y)[at] = __float2bfloat16(v);
  }
}

// Launch shapes.  A tile of few tokens can hold many adapters: with few tiles they are dealt out to
// 4 CTAs (dealt / not: 64 tokens with 60 adapters 26 / 46 us, 200 with 40 30 / 33, 500 with 60 39 / 35).
// With many tiles a CTA of the second product takes 512 columns, which share its set-up (4001 tokens
// 133 us, with 256 columns 140).
static int lora_deal(const LoraParams& p, int num_sms) {
  return p.tokens > 1 && (p.tokens + kLoraTile - 1) / kLoraTile < num_sms / 8 ? 4 : 1;
}

template <int NT>
static void launch_low(const LoraParams& p, int deal, cudaStream_t st) {
  launch_kernel(lora_low_kernel<NT, kLoraLowWarps, false>, dim3((p.tokens + kLoraTile - 1) / kLoraTile, p.low_parts, deal), kLoraLowWarps * 32,
                0, st, p);
}

template <int NT, int kWarps>
static cudaError_t launch_rows(const LoraParams& p, int num_sms, cudaStream_t st) {
  // CTAs that share a tile: while the GPU has room for more (three per SM) and each warp keeps 64 of k
  const int tiles = (p.tokens + kLoraTile - 1) / kLoraTile;
  unsigned share = 1;
  while (share < 8 && 2 * share * tiles <= 3u * num_sms && 2 * share * kWarps * 64 <= static_cast<unsigned>(p.k)) share *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = g_pdl_enabled ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = share;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles, share);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return cudaLaunchKernelEx(&cfg, lora_low_kernel<NT, kWarps, true>, p);
}

// the order of the tokens, then the rows of xs and the lists
cudaError_t launch_lora_rows(const LoraParams& p, int num_sms, cudaStream_t st) {
  launch_kernel(lora_sort_kernel, (p.tokens + 31) / 32, kLoraSortThreads, 0, st, p);
  cudaError_t e;
  if (p.rank <= 16) e = launch_rows<2, 8>(p, num_sms, st);
  else if (p.rank <= 32) e = launch_rows<4, 8>(p, num_sms, st);
  else if (p.rank <= 64) e = launch_rows<8, 8>(p, num_sms, st);
  else e = launch_rows<16, 4>(p, num_sms, st);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_lora(const LoraParams& p, int num_sms, cudaStream_t st) {
  const int deal = lora_deal(p, num_sms);
  if (p.order && !p.w) launch_kernel(lora_sort_kernel, (p.tokens + 31) / 32, kLoraSortThreads, 0, st, p);
  if (p.rank <= 16) launch_low<2>(p, deal, st);
  else if (p.rank <= 32) launch_low<4>(p, deal, st);
  else if (p.rank <= 64) launch_low<8>(p, deal, st);
  else launch_low<16>(p, deal, st);
  if (p.w) {   // few tokens
    const unsigned grid = (p.n + kLoraFewCols - 1) / kLoraFewCols;
    if (p.tokens <= 8) launch_kernel(lora_few_kernel<1>, grid, kLoraFewWarps * 32, 0, st, p);
    else launch_kernel(lora_few_kernel<2>, grid, kLoraFewWarps * 32, 0, st, p);
    return cudaGetLastError();
  }
  const int tiles = (p.tokens + kLoraTile - 1) / kLoraTile;
  const unsigned cols = (p.n + kLoraOutCols - 1) / kLoraOutCols;
  if (tiles >= num_sms) launch_kernel(lora_out_kernel<2>, dim3((cols + 1) / 2, tiles), kLoraOutWarps * 32, 0, st, p);
  else launch_kernel(lora_out_kernel<1>, dim3(cols, tiles, deal), kLoraOutWarps * 32, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2

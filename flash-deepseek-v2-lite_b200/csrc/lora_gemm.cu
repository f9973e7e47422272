// Shared projection and adapters of a long run of tokens (a prompt chunk) in one tcgen05 GEMM:
//   y[order[i], n] = bf16( sum_k xs[i, k] W[n, k] + sum_a sum_j L_a[i, j] B_a[n, j] )
// over tokens in adapter order (lora_sort_kernel): xs = the rows of x in that order, and
// L_a[i, j] = low[i, j] (fp32, in that order) where token i has adapter a, else 0.  A tile of 256 tokens holds few
// adapters, so their products are a few more steps of 64 k on the same accumulator (five against
// 32 at k = 2048 with five adapters of rank 32 in a tile), and neither the projection's fp32 sums nor
// the adapters' part ever reach memory: with separate launches those are 8 bytes written and read
// per output element.  The adapters' ranks are cut into pieces of 16, two to a step whatever
// adapters they belong to, and the steps stand evenly among the projection's: each is loaded while
// the ones before it are multiplied.
// low enters as the sum of two bf16 numbers (columns of their own against the same B), as in
// lora_out_kernel: 2^-16 of it is lost.  As one number it would lose 2^-8 of sum_j |low_j B_j|, far more than y's
// own rounding where terms cancel, and a token's precision would depend on how many share its call.
//
// A pair of SMs has a tile of 256 tokens x n_tile columns (tcgen05.mma on cta_group::2): each holds the
// operands and accumulators of 128 of the tokens and the operand of half of the columns, so that an SM
// brings in 128 + n_tile / 2 rows per step where a single SM with a 128 x n_tile tile brings in 128 +
// n_tile (all of the call 73 us, single SMs 75 us).  The issuing lanes are chosen by elect.sync: chosen
// by their number, each tcgen05.mma took some 200 clocks to issue and the GEMM 65 us instead of 46.
// Both operands K-major with the 128-byte swizzle, accumulators fp32 in TMEM, two of them.
// Persistent, one CTA per SM, 22 warps:
//  - warp 0 (one lane): TMA of this CTA's projection operands into a ring of 6 stages;
//  - warp 1 (one lane, of the pair's first CTA): tcgen05.mma for both;
//  - warps 2-5: accumulators to bf16 rows of y, while the next tile is multiplied;
//  - warps 6-21, in four groups that take the adapters' steps in turn: their operands, from global
//    memory through registers into ring stages; the loads are on their way before the stage is free.
//    (2 / 3 / 4 groups: 768 tokens with 64 adapters 47 / 44 / 40 us, 4001 with 6 71.4 / 72.0 / 72.2.  Rows of low and
//    B shared out over neighbouring lanes were slower: 52 / 49 / 47.)  A plain copy will not do: what an adapter's
//    padding past its rank holds must not be multiplied, nor may an infinity or a NaN of one adapter
//    meet the zeros that other adapters' tokens have in its columns.  Such values, and those of low, which would
//    meet the zeros that stand for them, enter as zeros, and the epilogue adds their products to the rows of
//    their own adapter.
// 4001 tokens, 6 adapters of rank 32, 2048 -> 3648: about 46 of the 71 us that the order, the rows and
// this take together; 1.3 PFLOP/s.  Bound by the multiplications with what the last tiles leave idle:
// 16 x 17 tiles are 3.7 rounds of 74 pairs.
#include "params.cuh"

namespace dsv2 {

constexpr int kLgK = 64;              // k of a ring stage
constexpr int kLgStages = 6;
constexpr int kLgStepPieces = kLgK / (2 * kLgPiece);   // pieces of an adapters' step, each with both parts of low
constexpr int kLgABytes = kLgRows * kLgK * 2;
constexpr int kLgMaxN = 256;
constexpr int kLgStageBytes = kLgABytes + kLgMaxN / 2 * kLgK * 2;
constexpr int kLgLoaders = 128;       // threads of a group that brings in the adapters' operands
constexpr int kLgGroups = 4;
constexpr int kLgThreads = 6 * 32 + kLgGroups * kLgLoaders;
constexpr size_t kLgSmem = kLgStages * kLgStageBytes + 1024 + 512;
static_assert(kLgSmem <= 232448, "adapter GEMM: shared memory exceeds 227 KB");

// The steps of an item: nkb of the projection and extra = ceil(pieces / 2) of the adapters, of which
// number e comes after (e + 1) nkb / (extra + 1) of the projection's.
struct LgSteps {
  int nkb, extra, kb, e, next;
  __device__ __forceinline__ LgSteps(int nkb_, int pieces)
      : nkb(nkb_), extra((pieces + kLgStepPieces - 1) / kLgStepPieces), kb(0), e(0), next(before(0)) {}
  __device__ __forceinline__ int before(int i) const { return static_cast<unsigned>((i + 1) * nkb) / static_cast<unsigned>(extra + 1); }
  __device__ __forceinline__ bool more() const { return kb < nkb || e < extra; }
  __device__ __forceinline__ bool adapters() const { return kb >= next && e < extra; }   // of the next step
  __device__ __forceinline__ void took_adapters() {   // (the division once for each of these, not for every step)
    ++e;
    next = before(e);
  }
};

// barrier 1 + group over a loader group; whether the predicate holds for all of it
__device__ __forceinline__ bool lg_all(int group, bool pred) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r)
               : "r"(static_cast<uint32_t>(pred)), "r"(1 + group), "r"(kLgLoaders)
               : "memory");
  return r != 0;
}
// arrive on a barrier of either CTA (cluster_addr)
__device__ __forceinline__ void lg_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// mbar_wait for arrivals from both CTAs
__device__ __forceinline__ bool lg_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_u32(bar)), "r"(parity)
                 : "memory");
    if (ok) return true;
  }
  set_device_error(kErrMbarTimeout);
  return false;
}
// a load into this CTA's shared memory that reports to a barrier of either
__device__ __forceinline__ void lg_tma(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(0)
      : "memory");
}
// true in one lane of the warp
__device__ __forceinline__ bool lg_elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void lg_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
               "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
// arrive on this barrier of both CTAs once every tcgen05.mma issued so far has completed
__device__ __forceinline__ void lg_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
__global__ __cluster_dims__(2, 1, 1) __launch_bounds__(kLgThreads, 1) void lora_gemm_kernel(
    const LoraParams p, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, int n_tile) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kLgStages * kLgStageBytes);   // (the first CTA's are used)
  uint64_t* empty_bar = full_bar + kLgStages;
  uint64_t* go_bar = empty_bar + kLgStages;       // [group][stage] the stage is free and that loader group's
  uint64_t* tfull_bar = go_bar + kLgGroups * kLgStages;   // [2]
  uint64_t* tempty_bar = tfull_bar + 2;           // [2] (the first CTA's)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_flag = abort_flag + 1;        // an adapter's B or low held an infinity or a NaN
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t half = cluster_ctarank();        // of the pair
  const int pair = cluster_id_x(), pairs = n_clusters_x();
  const int n_half = n_tile / 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kLgStages; ++s) {
      // the loads of both CTAs (announced by the first, which arrives twice) or the loaders of each
      mbar_init(&full_bar[s], 2);
      mbar_init(&empty_bar[s], 1);
      for (int q = 0; q < kLgGroups; ++q) mbar_init(&go_bar[q * kLgStages + s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 8);   // the epilogue warps of both
    }
    *abort_flag = 0;
    *odd_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive_release();
  cluster_wait_acquire();   // the other CTA's barriers are set up
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_enter();

  const int nkb = p.k / kLgK;
  const int m_tiles = (p.tokens + kLgM - 1) / kLgM, n_tiles = (p.n + n_tile - 1) / n_tile;
  const int items = m_tiles * n_tiles;
  // token tiles vary fastest: the pairs that run side by side share weight tiles
  auto list_of = [&](int mt) { return p.lists + mt * lg_list_ints(p.rank); };

  if (warp == 0) {
    // ---------------- TMA producer
    if (lg_elect()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int it = pair; it < items && !*abort_flag; it += pairs) {
        const int mt = it % m_tiles, nt = it / m_tiles;
        for (LgSteps q(nkb, list_of(mt)[0]); q.more();) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1)) {
            *abort_flag = 1;
            break;
          }
          if (q.adapters()) {
            // handed to the group whose step it is, by a barrier of its own: a wait for a parity is only
            // good for the next phase, so nobody may wait on a barrier some of whose phases they skip
            mbar_arrive(&go_bar[q.e % kLgGroups * kLgStages + stage]);
            q.took_adapters();
          } else {
            unsigned char* st = smem + stage * kLgStageBytes;
            if (half == 0) {
              mbar_arrive_expect_tx(&full_bar[stage], 2 * (kLgABytes + n_half * kLgK * 2));
              mbar_arrive(&full_bar[stage]);
            }
            const uint32_t bar = cluster_addr(&full_bar[stage], 0);
            lg_tma(smem_u32(st), &tmap_x, bar, q.kb * kLgK, mt * kLgM + half * kLgRows);
            lg_tma(smem_u32(st + kLgABytes), &tmap_w, bar, q.kb * kLgK, nt * n_tile + half * n_half);
            ++q.kb;
          }
          if (++stage == kLgStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer
    if (half == 0 && lg_elect()) {
      const uint32_t idesc = make_idesc_bf16(kLgM, n_tile);
      int stage = 0;
      uint32_t phase = 0, local = 0;
      for (int it = pair; it < items && !*abort_flag; it += pairs, ++local) {
        const int mt = it % m_tiles;
        const uint32_t buf = local & 1, use = local >> 1;
        if (!lg_wait(&tempty_bar[buf], (use & 1) ^ 1)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t dacc = tmem_base + buf * kLgMaxN;
        bool ok = true;
        const int pieces = list_of(mt)[0];
        bool first = true;
        for (LgSteps q(nkb, pieces); q.more();) {
          if (!lg_wait(&full_bar[stage], phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const bool ad = q.adapters();
          const int k16 = ad ? 2 * min(pieces - q.e * kLgStepPieces, kLgStepPieces) : kLgK / kLgPiece;
          unsigned char* st = smem + stage * kLgStageBytes;
          const uint64_t da = sw128_kmajor_desc(smem_u32(st)), db = sw128_kmajor_desc(smem_u32(st + kLgABytes));
          // adapters: columns 0-15 and 16-31 of A are a piece's high and low parts, both against columns 0-15 of B
          const int b1 = ad ? 0 : 2, b2 = ad ? 2 : 4, b3 = ad ? 2 : 6;
          lg_mma(dacc, da, db, idesc, first ? 0u : 1u);
          lg_mma(dacc, da + 2, db + b1, idesc, 1);
          if (k16 > 2) {
            lg_mma(dacc, da + 4, db + b2, idesc, 1);
            lg_mma(dacc, da + 6, db + b3, idesc, 1);
          }
          first = false;
          lg_commit(&empty_bar[stage]);
          if (++stage == kLgStages) {
            stage = 0;
            phase ^= 1;
          }
          if (ad) q.took_adapters();
          else ++q.kb;
        }
        if (!ok) {
          *abort_flag = 1;
          break;
        }
        lg_commit(&tfull_bar[buf]);
      }
    }
  } else if (warp < 6) {
    // ---------------- epilogue: lane = token, 16 columns at a time
    const int quad = warp & 3;
    uint32_t local = 0;
    for (int it = pair; it < items; it += pairs, ++local) {
      const int mt = it % m_tiles, nt = it / m_tiles;
      const int pos = mt * kLgM + half * kLgRows + quad * 32 + lane;
      const bool live = pos < p.tokens;
      bf16* y = static_cast<bf16*>(p.y) + (live ? p.order[pos] : 0) * p.y_row_stride + nt * n_tile;
      const uint32_t buf = local & 1, use = local >> 1;
      const bool ok = lg_wait(&tfull_bar[buf], use & 1);
      if (!ok || *abort_flag) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t tbase = tmem_base + buf * kLgMaxN + (static_cast<uint32_t>(quad * 32) << 16);
      const int cols = min(n_tile, p.n - nt * n_tile);
      for (int c = 0; c < n_tile; c += 32) {
        float v[2][16];
        tmem_ld16(tbase + c, v[0]);
        tmem_ld16(tbase + c + 16, v[1]);
        tmem_ld_wait();
        if (live) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float* a = &v[h >> 1][8 * (h & 1)];
            if (c + 8 * h < cols)
              *reinterpret_cast<uint4*>(y + c + 8 * h) =
                  make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) lg_arrive(cluster_addr(&tempty_bar[buf], 0));
      if (*odd_flag && live && p.order[p.tokens + pos] >= 0) {
        // the products that were left out, into this thread's own elements of y (rare: any speed will do)
        const int a = p.order[p.tokens + pos], rank = p.order[2 * p.tokens + pos];
        const float* low = p.low + static_cast<long long>(pos) * p.rank;
        const bf16* b = p.b + (static_cast<long long>(a) * p.n + nt * n_tile) * p.rank;
        for (int c = 0; c < cols; ++c, b += p.rank)
          for (int j = 0; j < rank; ++j) {
            const float w = __bfloat162float(b[j]), l = low[j];
            if (isfinite(w) && isfinite(__bfloat162float(__float2bfloat16(l)))) continue;
            y[c] = __float2bfloat16(__bfloat162float(y[c]) + l * w);
          }
      }
    }
  } else {
    // ---------------- adapters' operands: thread = token row of A and row of B
    const int group = (warp - 6) / (kLgLoaders / 32);
    const int t = threadIdx.x - 6 * 32 - group * kLgLoaders;
    int stage = 0;
    uint32_t go_phase = 0;   // bit s: parity of the group's next use of stage s
    bool ok = true;
    for (int it = pair; it < items && ok; it += pairs) {
      const int mt = it % m_tiles, nt = it / m_tiles;
      const int pos = mt * kLgM + half * kLgRows + t;
      const int mine = pos < p.tokens ? p.order[p.tokens + pos] : -1;
      const float* low = p.low + static_cast<long long>(min(pos, p.tokens - 1)) * p.rank;
      const int* list = list_of(mt);
      const int n = nt * n_tile + half * n_half + t;
      const bool in = t < n_half && n < p.n;
      const int pieces = list[0];
      LgSteps q(nkb, pieces);
      int done = 0;   // steps of this item before the next adapters' one
      for (; q.e < q.extra && ok; q.took_adapters()) {
        const int at = q.next + q.e;   // of the item's steps
        stage = (stage + at - done) % kLgStages;
        done = at + 1;
        const int st_i = stage;
        stage = (stage + 1) % kLgStages;
        if (q.e % kLgGroups != group) continue;   // another group's
        const uint32_t parity = (go_phase >> st_i) & 1;
        go_phase ^= 1u << st_i;
        constexpr int kChunks = 2 * kLgStepPieces;   // of 8 ranks
        uint4 ra[kChunks], rl[kChunks], rb[kChunks];   // low's two parts (at first its 8 fp32 numbers), B
        int2 u[kLgStepPieces];   // this step's pieces; none: no ranks
#pragma unroll
        for (int g = 0; g < kLgStepPieces; ++g) {
          const int piece = q.e * kLgStepPieces + g;
          u[g] = piece < pieces ? __ldg(reinterpret_cast<const int2*>(list + 2 + 2 * piece)) : make_int2(0, 0);
        }
        // no branches here: all of a step's loads are under way together
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int a = u[c >> 1].x, j = (u[c >> 1].y & 0xffff) + 8 * (c & 1), left = (u[c >> 1].y >> 16) - 8 * (c & 1);
          ra[c] = ld_or_zero(low + j, mine == a && left > 0);
          rl[c] = ld_or_zero(low + j + 4, mine == a && left > 0);
          rb[c] = ld_or_zero(p.b + (static_cast<long long>(a) * p.n + n) * p.rank + j, in && left > 0);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int left = (u[c >> 1].y >> 16) - 8 * (c & 1);
          if (left <= 0 || left >= 8) continue;
          // padding past the rank may be anything, and 0 * NaN is not 0
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t keep = 2 * i >= left ? 0u : 2 * i + 1 >= left ? 0xffffu : 0xffffffffu;
            reinterpret_cast<uint32_t*>(&rb[c])[i] &= keep;
          }
        }
        bool odd = false;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          odd |= drop_nonfinite(rb[c]);
          const uint32_t w[8] = {ra[c].x, ra[c].y, ra[c].z, ra[c].w, rl[c].x, rl[c].y, rl[c].z, rl[c].w};
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v0 = __uint_as_float(w[2 * i]), v1 = __uint_as_float(w[2 * i + 1]);
            hi[i] = pack_bf16x2(v0, v1);
            lo[i] = pack_bf16x2(v0 - bf16lo(hi[i]), v1 - bf16hi(hi[i]));
          }
          ra[c] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          rl[c] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          if (drop_nonfinite(ra[c])) {   // (what is left of an infinity or a NaN is not finite either)
            drop_nonfinite(rl[c]);
            odd = true;
          }
        }
        if (odd)
          for (uint32_t r = 0; r < 2; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(const_cast<int*>(odd_flag), r)), "r"(1) : "memory");
        if (mbar_wait(&go_bar[group * kLgStages + st_i], parity)) {
          unsigned char* st = smem + st_i * kLgStageBytes;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const int at = 4 * (c >> 1) + (c & 1);
            *reinterpret_cast<uint4*>(st + swz(t, at)) = ra[c];
            *reinterpret_cast<uint4*>(st + swz(t, at + 2)) = rl[c];
            if (t < n_half) *reinterpret_cast<uint4*>(st + kLgABytes + swz(t, c)) = rb[c];
          }
          fence_proxy_async_smem();
        } else {
          *abort_flag = 1;
          ok = false;
        }
        __syncwarp();
        ok = lg_all(group, ok);   // all of the group go on, or none
        if (ok && t == 0) lg_arrive(cluster_addr(&full_bar[st_i], 0));
      }
      stage = (stage + nkb + q.extra - done) % kLgStages;
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_arrive_release();
  cluster_wait_acquire();   // neither CTA's shared memory or TMEM is used any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

cudaError_t lora_gemm_init() {
  return cudaFuncSetAttribute(lora_gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLgSmem));
}

// Columns of a tile: the width that leaves the least operand traffic in the longest-running pair (tiles
// are dealt out evenly; per step an SM brings in 128 + n_tile / 2 rows).
int lora_gemm_tile(int tokens, int n, int num_sms) {
  const long long m_tiles = (tokens + kLgM - 1) / kLgM, pairs = num_sms / 2;
  long long best = -1;
  int tile = kLgMaxN;
  for (int c = kLgMaxN; c >= 64; c -= 32) {
    const long long rounds = (m_tiles * ((n + c - 1) / c) + pairs - 1) / pairs, cost = rounds * (kLgRows + c / 2);
    if (best < 0 || cost < best) {
      best = cost;
      tile = c;
    }
  }
  return tile;
}

cudaError_t launch_lora_gemm(const LoraParams& p, const CUtensorMap& tm_x, const CUtensorMap& tm_w, int n_tile, int num_sms,
                             cudaStream_t st) {
  const long long items = static_cast<long long>((p.tokens + kLgM - 1) / kLgM) * ((p.n + n_tile - 1) / n_tile);
  launch_kernel(lora_gemm_kernel, 2 * static_cast<unsigned>(std::min<long long>(items, num_sms / 2)), kLgThreads, kLgSmem, st, p, tm_x, tm_w,
                n_tile);
  return cudaGetLastError();
}

}  // namespace dsv2

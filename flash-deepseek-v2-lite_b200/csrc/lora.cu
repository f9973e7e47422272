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

// order[pos] = t with pos = #{u: id_u < id_t} + #{u < t: id_u = id_t}: every pair of tokens is
// compared once, 16 million at 4096 tokens (about 2 us over the GPU), with no histogram over the
// adapters, whose number is the caller's.
__global__ __launch_bounds__(256) void lora_sort_kernel(const LoraParams p) {
  pdl_enter();
  __shared__ int s_id[256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // 8 warps share a group of 32 tokens: lane = token, warp = an eighth of the others
  const int t = blockIdx.x * 32 + lane;
  const int mine = t < p.tokens ? lora_id(p, t) : 0;
  int before = 0;
  for (int u0 = 0; u0 < p.tokens; u0 += 256) {
    __syncthreads();
    const int u = u0 + threadIdx.x;
    s_id[threadIdx.x] = u < p.tokens ? lora_id(p, u) : 0x7fffffff;
    __syncthreads();
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
      const int v = s_id[warp * 32 + i];
      before += (v < mine || (v == mine && u0 + warp * 32 + i < t)) ? 1 : 0;
    }
  }
  __syncthreads();
  s_id[threadIdx.x] = before;
  __syncthreads();
  if (warp == 0 && t < p.tokens) {
    for (int w = 1; w < 8; ++w) before += s_id[w * 32 + lane];
    p.order[before] = t;
  }
}

// The 16 tokens of tile i and their adapters, in shared memory; -2 marks a place without a token.
__device__ __forceinline__ void lora_tile(const LoraParams& p, int tile, int* s_tok, int* s_ad) {
  if (threadIdx.x < kLoraTile) {
    const int i = tile * kLoraTile + threadIdx.x;
    const int t = i < p.tokens ? (p.order ? p.order[i] : i) : -1;
    s_tok[threadIdx.x] = t;
    s_ad[threadIdx.x] = t >= 0 ? lora_id(p, t) : -2;
  }
  __syncthreads();
}

// next adapter above `last` in the tile, or a large number
__device__ __forceinline__ int lora_next(const int* s_ad, int last) {
  int a = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kLoraTile; ++i) {
    const int v = s_ad[i];
    if (v > last) a = min(a, v);
  }
  return a;
}

__device__ __forceinline__ uint4 ld_or_zero(const void* q, bool in) {
  return in ? __ldg(reinterpret_cast<const uint4*>(q)) : make_uint4(0, 0, 0, 0);
}

// low partials of one tile and k split: low[split, t, j].  NT = rank / 8 n-tiles of 8 ranks.
template <int NT>
__global__ __launch_bounds__(kLoraLowWarps * 32) void lora_low_kernel(const LoraParams p) {
  pdl_enter();
  __shared__ int s_tok[kLoraTile], s_ad[kLoraTile];
  __shared__ float s_sum[kLoraLowWarps][kLoraTile][8 * NT + 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  lora_tile(p, blockIdx.x, s_tok, s_ad);
  // this CTA's k range, in steps of 32, and this warp's part of it
  const int steps = (p.k + 31) / 32, splits = gridDim.y * kLoraLowWarps, part = blockIdx.y * kLoraLowWarps + warp;
  const int k0 = static_cast<int>(static_cast<long long>(steps) * part / splits) * 32;
  const int k1 = static_cast<int>(static_cast<long long>(steps) * (part + 1) / splits) * 32;
  const int t0 = s_tok[gq], t1 = s_tok[gq + 8];
  const bf16* x0 = p.x + (t0 >= 0 ? t0 : 0) * p.x_row_stride;
  const bf16* x1 = p.x + (t1 >= 0 ? t1 : 0) * p.x_row_stride;
  for (int a = lora_next(s_ad, -1); a != 0x7fffffff; a = lora_next(s_ad, a)) {
    const bf16* w = p.a + static_cast<long long>(a) * p.rank * p.k;
    const int rank = min(max(p.ranks[a], 0), p.rank), nt = (rank + 7) / 8;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const bool m0 = s_ad[gq] == a, m1 = s_ad[gq + 8] == a;
#pragma unroll 2
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
    __syncthreads();   // the previous adapter's sums have been read
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s_sum[warp][gq][8 * n + 2 * tq] = acc[n][0];
      s_sum[warp][gq][8 * n + 2 * tq + 1] = acc[n][1];
      s_sum[warp][gq + 8][8 * n + 2 * tq] = acc[n][2];
      s_sum[warp][gq + 8][8 * n + 2 * tq + 1] = acc[n][3];
    }
    __syncthreads();
    const float scale = p.scales[a];
    for (int i = threadIdx.x; i < kLoraTile * 8 * NT; i += kLoraLowWarps * 32) {
      const int r = i / (8 * NT), j = i % (8 * NT);
      if (s_ad[r] != a || j >= p.rank) continue;
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kLoraLowWarps; ++q) v += s_sum[q][r][j];
      // columns past the adapter's rank hold whatever its padding holds
      p.low[(static_cast<long long>(blockIdx.y) * p.tokens + s_tok[r]) * p.rank + j] = j < rank ? v * scale : 0.f;
    }
  }
}

// y tile: 16 tokens x 256 columns.  A warp owns 32 columns as two pairs of n-tiles; column 2 q + e of
// n-tile u of a pair is column 4 q + 2 u + e of its 16, so that a lane ends with 4 consecutive
// columns: whole sectors of the partials in, of y out.  low is used as the sum of two bf16 numbers
// (16 significant bits), so that it adds no rounding of its own to y.
__global__ __launch_bounds__(kLoraOutWarps * 32) void lora_out_kernel(const LoraParams p) {
  pdl_enter();
  __shared__ int s_tok[kLoraTile], s_ad[kLoraTile];
  __shared__ __align__(16) uint32_t s_hi[kLoraTile][68], s_lo[kLoraTile][68];   // bf16 pairs, up to 128 ranks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  lora_tile(p, blockIdx.y, s_tok, s_ad);
  // the tile's low rows: the k splits summed in order, as high and low bf16 parts; 0 past the rank
  const int pairs = (p.rank + 31) / 32 * 16;
  for (int i = threadIdx.x; i < kLoraTile * pairs; i += kLoraOutWarps * 32) {
    const int r = i / pairs, j = 2 * (i % pairs);
    float v0 = 0.f, v1 = 0.f;
    if (s_ad[r] >= 0 && j < p.rank) {
      for (int q = 0; q < p.low_parts; ++q) {
        const float2 v = *reinterpret_cast<const float2*>(p.low + (static_cast<long long>(q) * p.tokens + s_tok[r]) * p.rank + j);
        v0 += v.x;
        v1 += v.y;
      }
    }
    const uint32_t hi = pack_bf16x2(v0, v1);
    s_hi[r][i % pairs] = hi;
    s_lo[r][i % pairs] = pack_bf16x2(v0 - bf16lo(hi), v1 - bf16hi(hi));
  }
  const int n0 = blockIdx.x * kLoraOutCols + warp * 32;
  const int t0 = s_tok[gq], t1 = s_tok[gq + 8];
  float acc[4][4];   // n-tiles 0, 1: columns n0 .. + 16; 2, 3: + 16 .. + 32
#pragma unroll
  for (int u = 0; u < 4; ++u) acc[u][0] = acc[u][1] = acc[u][2] = acc[u][3] = 0.f;
  // shared projection: 4 consecutive columns of two tokens per pair
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = n0 + 16 * h + 4 * tq;
    if (n >= p.n) continue;
    for (int q = 0; q < p.base_parts; ++q) {
      const float* b = p.base + q * p.base_part_stride + n;
      if (t0 >= 0) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(b + t0 * p.base_row_stride));
        acc[2 * h][0] += v.x;
        acc[2 * h][1] += v.y;
        acc[2 * h + 1][0] += v.z;
        acc[2 * h + 1][1] += v.w;
      }
      if (t1 >= 0) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(b + t1 * p.base_row_stride));
        acc[2 * h][2] += v.x;
        acc[2 * h][3] += v.y;
        acc[2 * h + 1][2] += v.z;
        acc[2 * h + 1][3] += v.w;
      }
    }
  }
  __syncthreads();
  for (int a = lora_next(s_ad, -1); a != 0x7fffffff; a = lora_next(s_ad, a)) {
    const int rank = min(max(p.ranks[a], 0), p.rank);
    const bool m0 = s_ad[gq] == a, m1 = s_ad[gq + 8] == a;
    for (int j = 0; j < rank; j += 32) {
      // lane tq takes ranks j + 8 tq .. + 8 (4 words of the staged pairs)
      const int jw = j / 2 + 4 * tq;
      uint4 h0 = make_uint4(0, 0, 0, 0), h1 = h0, l0 = h0, l1 = h0;
      if (m0) {
        h0 = *reinterpret_cast<const uint4*>(&s_hi[gq][jw]);
        l0 = *reinterpret_cast<const uint4*>(&s_lo[gq][jw]);
      }
      if (m1) {
        h1 = *reinterpret_cast<const uint4*>(&s_hi[gq + 8][jw]);
        l1 = *reinterpret_cast<const uint4*>(&s_lo[gq + 8][jw]);
      }
      const uint32_t ah0[4] = {h0.x, h1.x, h0.y, h1.y}, ah1[4] = {h0.z, h1.z, h0.w, h1.w};
      const uint32_t al0[4] = {l0.x, l1.x, l0.y, l1.y}, al1[4] = {l0.z, l1.z, l0.w, l1.w};
      const int mine = rank - j - 8 * tq;   // ranks of this lane's 8 that exist
      uint4 b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int n = n0 + 16 * (u >> 1) + 4 * (gq >> 1) + 2 * (u & 1) + (gq & 1);
        b[u] = ld_or_zero(p.b + (static_cast<long long>(a) * p.n + n) * p.rank + j + 8 * tq, n < p.n && mine > 0);
        if (mine > 0 && mine < 8) {
          // padding past the rank may be anything, and 0 * NaN is not 0
          uint32_t* bw = reinterpret_cast<uint32_t*>(&b[u]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (2 * i >= mine) bw[i] = 0;
            else if (2 * i + 1 >= mine) bw[i] &= 0xffffu;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        mma_bf16_16816(acc[u], ah0, b[u].x, b[u].y);
        mma_bf16_16816(acc[u], al0, b[u].x, b[u].y);
        mma_bf16_16816(acc[u], ah1, b[u].z, b[u].w);
        mma_bf16_16816(acc[u], al1, b[u].z, b[u].w);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = n0 + 16 * h + 4 * tq;
    if (n >= p.n) continue;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int t = c ? t1 : t0;
      if (t < 0) continue;
      const float v0 = acc[2 * h][2 * c], v1 = acc[2 * h][2 * c + 1], v2 = acc[2 * h + 1][2 * c], v3 = acc[2 * h + 1][2 * c + 1];
      const long long off = t * p.y_row_stride + n;
      if (p.y_f32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.y) + off) = make_float4(v0, v1, v2, v3);
      else *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(p.y) + off) = make_uint2(pack_bf16x2(v0, v1), pack_bf16x2(v2, v3));
    }
  }
}

cudaError_t launch_lora(const LoraParams& p, cudaStream_t st) {
  const int tiles = (p.tokens + kLoraTile - 1) / kLoraTile;
  if (p.order) launch_kernel(lora_sort_kernel, (p.tokens + 31) / 32, 256, 0, st, p);
  const dim3 grid(tiles, p.low_parts), block(kLoraLowWarps * 32);
  if (p.rank <= 16) launch_kernel(lora_low_kernel<2>, grid, block, 0, st, p);
  else if (p.rank <= 32) launch_kernel(lora_low_kernel<4>, grid, block, 0, st, p);
  else if (p.rank <= 64) launch_kernel(lora_low_kernel<8>, grid, block, 0, st, p);
  else launch_kernel(lora_low_kernel<16>, grid, block, 0, st, p);
  launch_kernel(lora_out_kernel, dim3((p.n + kLoraOutCols - 1) / kLoraOutCols, tiles), kLoraOutWarps * 32, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2

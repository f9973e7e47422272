// Low-rank adapters of many requests beside a shared projection:
//   low[t, j] = scale_a * sum_k x[t, k] A_a[j, k]           (fp32, j < rank of a)
//   y[t, n]   = sum of the shared projection's partials + sum_j low[t, j] B_a[n, j]
// with a = the adapter of token t (none: y is the shared projection alone).
#include "params.cuh"

namespace dsv2 {

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
  return a;
}

__global__ __launch_bounds__(256) void lora_low_simple_kernel(const LoraParams p) {
  pdl_enter();
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int a = lora_id(p, t);
  if (a < 0) return;
  const int rank = min(max(p.ranks[a], 0), p.rank);
  const bf16* x = p.x + t * p.x_row_stride;
  for (int j = warp; j < rank; j += 8) {
    const bf16* w = p.a + (static_cast<long long>(a) * p.rank + j) * p.k;
    float s = 0.f;
    for (int k = 8 * lane; k < p.k; k += 256)
      s = dot8(*reinterpret_cast<const uint4*>(x + k), *reinterpret_cast<const uint4*>(w + k), s);
    s = warp_sum(s);
    if (lane == 0) p.low[static_cast<long long>(t) * p.rank + j] = s * p.scales[a];
  }
}

__global__ __launch_bounds__(256) void lora_expand_simple_kernel(const LoraParams p) {
  pdl_enter();
  const int t = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  const int a = lora_id(p, t);
  if (n >= p.n) return;
  float s = 0.f;
  for (int i = 0; i < p.base_parts; ++i) s += p.base[i * p.base_part_stride + t * p.base_row_stride + n];
  if (a >= 0) {
    const int rank = min(max(p.ranks[a], 0), p.rank);
    const bf16* b = p.b + (static_cast<long long>(a) * p.n + n) * p.rank;
    const float* low = p.low + static_cast<long long>(t) * p.rank;
    for (int j = 0; j < rank; ++j) s = fmaf(low[j], __bfloat162float(b[j]), s);
  }
  const long long off = t * p.y_row_stride + n;
  if (p.y_f32) reinterpret_cast<float*>(p.y)[off] = s;
  else reinterpret_cast<bf16*>(p.y)[off] = __float2bfloat16_rn(s);
}

cudaError_t launch_lora(const LoraParams& p, cudaStream_t st) {
  launch_kernel(lora_low_simple_kernel, p.tokens, 256, 0, st, p);
  launch_kernel(lora_expand_simple_kernel, dim3((p.n + 255) / 256, p.tokens), 256, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2

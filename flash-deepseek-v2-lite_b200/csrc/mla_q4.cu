// Latent attention over the paged 4-bit cache (latent4.cuh):
//   score[h, s] = scale * (q_abs[h] . latent[s] + q_pe[h] . rope[s]),  s = 0 .. position
//   o_lat[h]    = sum_s softmax(score)[h, s] * latent[s]
// for the 16 heads of every query row; the tokens of a row come from the pages of its
// block-table row.  One CTA per query row, one warp per head, one 16-token block at a time.
#include "latent4.cuh"
#include "params.cuh"

namespace dsv2 {

__global__ __launch_bounds__(512) void mla_q4_simple_kernel(const MlaQ4Params p) {
  pdl_enter();
  __shared__ bf16 s_tok[kL4Tokens][578];   // every value is exact in bf16
  __shared__ bf16 s_q[kHeads][578];
  const int tid = threadIdx.x, lane = tid & 31, h = tid >> 5;
  const int row = blockIdx.x;
  const long long pos = p.positions[row];
  const int seq = p.seq_rows ? p.seq_rows[row] : row;
  long long len = (seq < 0 || pos < 0) ? 0 : pos + 1;
  if (len > 0 && (seq >= p.seqs || len > static_cast<long long>(p.width) * p.page_blocks * kL4Tokens)) {
    if (tid == 0) set_device_error(kErrIndex);
    len = 0;
  }
  for (int i = tid; i < kHeads * 512; i += 512) s_q[i >> 9][i & 511] = p.q_abs[static_cast<long long>(row) * kHeads * 512 + i];
  for (int i = tid; i < kHeads * 64; i += 512) s_q[i >> 6][512 + (i & 63)] = p.q_pe[static_cast<long long>(row) * kHeads * 64 + i];
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
  for (long long b = 0; b * kL4Tokens < len; ++b) {
    long long blk = p.table[seq * p.table_stride + b / p.page_blocks] * static_cast<long long>(p.page_blocks) + b % p.page_blocks;
    if (blk < 0 || blk >= p.n_blocks) {
      if (tid == 0) set_device_error(kErrIndex);
      blk = 0;
    }
    const unsigned char* src = p.cache + blk * kL4BlockBytes;
    __syncthreads();
    for (int i = tid; i < kL4Tokens * 64; i += 512) {
      const int t = i >> 6, w = i & 63;
      float x[8];
      l4_unpack(*reinterpret_cast<const uint32_t*>(src + l4_word_off(t, w >> 2, w & 3)),
                l4_scale(src[kL4ScaleOff + 16 * (w >> 2) + l4_scale_place(t)]), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) s_tok[t][8 * w + j] = __float2bfloat16_rn(x[j]);
    }
    {
      const int t = tid >> 5, r = lane;
      const uint32_t u = *reinterpret_cast<const uint32_t*>(src + l4_rope_off(t, r));
      *reinterpret_cast<uint32_t*>(&s_tok[t][512 + 2 * r]) = u;
    }
    __syncthreads();
    const int n = static_cast<int>(min(static_cast<long long>(kL4Tokens), len - b * kL4Tokens));
    for (int t = 0; t < n; ++t) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 18; ++j) s = fmaf(__bfloat162float(s_q[h][lane + 32 * j]), __bfloat162float(s_tok[t][lane + 32 * j]), s);
      s = warp_sum(s) * p.scale_log2;
      const float mn = fmaxf(m, s), u = mn == -INFINITY ? 0.f : mn;
      const float a = exp2f(m - u), e = exp2f(s - u);
      l = l * a + e;
      m = mn;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = o[i] * a + e * __bfloat162float(s_tok[t][lane + 32 * i]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bf16* out = p.o_lat + (static_cast<long long>(row) * kHeads + h) * 512;
#pragma unroll
  for (int i = 0; i < 16; ++i) out[lane + 32 * i] = __float2bfloat16_rn(o[i] * inv);
}

cudaError_t launch_mla_q4(const MlaQ4Params& p, cudaStream_t st) {
  launch_kernel(mla_q4_simple_kernel, p.rows, 512, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2

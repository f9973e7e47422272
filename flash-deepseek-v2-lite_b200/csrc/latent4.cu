// Rows of the 4-bit latent cache (latent4.cuh): quantise-and-scatter by slot, and the read-back
// of the values they stand for.  Both are bound by memory: 1152 bytes of bf16 row and 400 of
// cache per token, each moved once.  One warp per token: lane l owns dims [16 l, 16 l + 16),
// half of a group, so a group's maximum is one shuffle away and a token's 256 packed bytes
// leave as one contiguous segment.  16381 tokens: write 11.3 us (2.3 TB/s), read 5.6 us (4.6 TB/s);
// one token 2.7 and 1.4 us.
#include "latent4.cuh"
#include "params.cuh"

namespace dsv2 {

constexpr int kL4Warps = 4;   // tokens per CTA

__global__ __launch_bounds__(kL4Warps * 32) void latent4_write_kernel(const Latent4Params p) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * kL4Warps + (threadIdx.x >> 5);
  if (t >= p.n) return;
  const long long slot = p.slots[t];
  if (slot < 0) return;                                  // padding
  if (slot >= p.n_blocks * kL4Tokens) {
    if (lane == 0) set_device_error(kErrIndex);
    return;
  }
  const bf16* row = p.rows + t * p.row_stride;
  const uint4 u0 = *reinterpret_cast<const uint4*>(row + 16 * lane);
  const uint4 u1 = *reinterpret_cast<const uint4*>(row + 16 * lane + 8);
  const uint32_t rope = *reinterpret_cast<const uint32_t*>(row + kL4Groups * 32 + 2 * lane);
  const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
  float x[2][8];
  float amax = 0.f;
  bool bad = l4_nonfinite(rope);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float lo = bf16lo(w[i]), hi = bf16hi(w[i]);
    x[i >> 2][2 * (i & 3)] = lo;
    x[i >> 2][2 * (i & 3) + 1] = hi;
    amax = fmaxf(amax, fmaxf(fabsf(lo), fabsf(hi)));     // fmaxf drops a NaN
    bad |= l4_nonfinite(w[i]);
  }
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  const int code = l4_code(amax);
  const float scale = l4_scale(code);
  const int tok = static_cast<int>(slot & (kL4Tokens - 1)), g = lane >> 1;
  unsigned char* blk = p.cache + (slot >> 4) * kL4BlockBytes;
  *reinterpret_cast<uint2*>(blk + l4_word_off(tok, g, 2 * (lane & 1))) = make_uint2(l4_pack(x[0], scale), l4_pack(x[1], scale));
  if ((lane & 1) == 0) blk[kL4ScaleOff + 16 * g + l4_scale_place(tok)] = static_cast<unsigned char>(code);
  *reinterpret_cast<uint32_t*>(blk + l4_rope_off(tok, lane)) = rope;
  if (bad) set_device_error(kErrNonFinite);
}

__global__ __launch_bounds__(kL4Warps * 32) void latent4_read_kernel(const Latent4Params p) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * kL4Warps + (threadIdx.x >> 5);
  if (t >= p.n) return;
  const long long slot = p.slots[t];
  bf16* row = p.out + t * p.row_stride;
  uint4 o0 = make_uint4(0, 0, 0, 0), o1 = o0;
  uint32_t rope = 0;
  const bool in = slot >= 0 && slot < p.n_blocks * kL4Tokens;
  if (in) {
    const int tok = static_cast<int>(slot & (kL4Tokens - 1)), g = lane >> 1;
    const unsigned char* blk = p.cache + (slot >> 4) * kL4BlockBytes;
    const uint2 w = *reinterpret_cast<const uint2*>(blk + l4_word_off(tok, g, 2 * (lane & 1)));
    const float scale = l4_scale(blk[kL4ScaleOff + 16 * g + l4_scale_place(tok)]);
    rope = *reinterpret_cast<const uint32_t*>(blk + l4_rope_off(tok, lane));
    float x[8];
    l4_unpack(w.x, scale, x);
    o0 = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    l4_unpack(w.y, scale, x);
    o1 = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  } else if (slot >= 0 && lane == 0) {
    set_device_error(kErrIndex);
  }
  *reinterpret_cast<uint4*>(row + 16 * lane) = o0;       // padding reads as zeros
  *reinterpret_cast<uint4*>(row + 16 * lane + 8) = o1;
  *reinterpret_cast<uint32_t*>(row + kL4Groups * 32 + 2 * lane) = rope;
}

cudaError_t launch_latent4_write(const Latent4Params& p, cudaStream_t st) {
  launch_kernel(latent4_write_kernel, static_cast<unsigned>((p.n + kL4Warps - 1) / kL4Warps), kL4Warps * 32, 0, st, p);
  return cudaGetLastError();
}

cudaError_t launch_latent4_read(const Latent4Params& p, cudaStream_t st) {
  launch_kernel(latent4_read_kernel, static_cast<unsigned>((p.n + kL4Warps - 1) / kL4Warps), kL4Warps * 32, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2

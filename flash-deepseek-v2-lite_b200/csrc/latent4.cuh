// The 4-bit latent cache: 16-token blocks of 6400 bytes (400 bytes a token instead of the 1152
// of the bf16 latent cache).  A cache is an array of such blocks; slot s is token s % 16 of
// block s / 16, and a page is page_size / 16 consecutive blocks.
//
//   [0, 4096)     token p at 256 p: 16 groups of 32 latent dims, 16 bytes each; group c sits at
//                 place c ^ l4_group_xor(p).  Word w of a group holds dims 8w .. 8w + 7: dim
//                 8w + 2i in nibble i and dim 8w + 2i + 1 in nibble 4 + i, each as v + 8 with
//                 v in -8 .. 7; the element is v * scale
//   [4096, 4352)  scale codes: group c of token p at 4096 + 16 c + l4_scale_place(p)
//   [4352, 6400)  roped key dims, bf16: token p at 4352 + 128 p, chunk j (8 dims) at j ^ (p & 4)
//
// Scale: max |x| of the group / 7, rounded to nearest even at 3 mantissa bits; the code is bits
// 14..7 of the scale as a positive fp16 number (5 exponent bits, 3 mantissa bits), so decoding
// is one shift.  v = round(x / scale).  A scale has 4 significant bits and v four, so every
// value has at most 8: exact in bf16 and in fp16.  Codes end at 167, scale 60 (groups beyond
// 60 * 7 saturate); bytes of slots that were never written may decode to an infinity or NaN.
//
// The places are the shared-memory layout of the attention kernel (mla_q4.cu): a block is
// copied as it lies, and the fragment loads of both products hit all 32 banks once.
//  * scores read 16 bytes (one group) per lane: the 8 lanes of a phase take tokens p, p + 4 and
//    four neighbouring groups; l4_group_xor(p) and l4_group_xor(p + 4) differ in bit 2;
//  * P V reads one word per lane: 4 tokens with p & 3 = 0..3 and two neighbouring groups;
//    l4_group_xor takes 4 values over them that differ in bits 1 and 2.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace dsv2 {

constexpr int kL4Tokens = 16;
constexpr int kL4Groups = 16;               // groups of 32 latent dims
constexpr int kL4BlockBytes = 6400;
constexpr int kL4ScaleOff = 4096;
constexpr int kL4RopeOff = 4352;
constexpr int kL4MaxCode = 167;             // scale 60

__device__ __forceinline__ int l4_group_xor(int p) { return 2 * (p & 1) + 4 * (((p >> 1) ^ (p >> 2)) & 1); }
__device__ __forceinline__ int l4_scale_place(int p) { return 4 * (p & 3) + (p >> 2); }

// byte offset in the block of word w (0..3) of group c of token p, and of rope word r (0..31: 2 dims)
__device__ __forceinline__ int l4_word_off(int p, int c, int w) { return p * 256 + ((c ^ l4_group_xor(p)) << 4) + 4 * w; }
__device__ __forceinline__ int l4_rope_off(int p, int r) { return kL4RopeOff + p * 128 + (((r >> 2) ^ (p & 4)) << 4) + 4 * (r & 3); }

__device__ __forceinline__ float l4_scale(int code) { return __half2float(__ushort_as_half(static_cast<unsigned short>(code << 7))); }

// Scale code of a group with largest magnitude amax (finite or infinite, not NaN).
__device__ __forceinline__ int l4_code(float amax) {
  const float s = __fdiv_rn(amax, 7.f);
  int code;
  if (s < 6.103515625e-5f) {          // below the smallest normal scale 2^-14: multiples of 2^-17
    code = __float2int_rn(s * 131072.f);
  } else {
    const int bits = __float_as_int(s);
    code = ((bits + 0x7ffff + ((bits >> 20) & 1)) >> 20) - (112 << 3);
  }
  return min(code, kL4MaxCode);
}

// v + 8 of one element; scale 0 (a group of zeros, or too small for any scale) gives 8.
// NaN has no nibble and becomes 0 (the caller raises the device error word).
__device__ __forceinline__ uint32_t l4_nibble(float x, float scale) {
  if (!(scale > 0.f) || x != x) return 8u;
  return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -8.f), 7.f)) + 8);
}

// word of 8 consecutive dims
__device__ __forceinline__ uint32_t l4_pack(const float (&x)[8], float scale) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w |= l4_nibble(x[2 * i], scale) << (4 * i);
    w |= l4_nibble(x[2 * i + 1], scale) << (16 + 4 * i);
  }
  return w;
}

// the 8 dims of a word
__device__ __forceinline__ void l4_unpack(uint32_t w, float scale, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = static_cast<float>(static_cast<int>((w >> (4 * i)) & 15u) - 8) * scale;
    x[2 * i + 1] = static_cast<float>(static_cast<int>((w >> (16 + 4 * i)) & 15u) - 8) * scale;
  }
}

__device__ __forceinline__ bool l4_nonfinite(uint32_t bf16x2) {
  return (bf16x2 & 0x7f80u) == 0x7f80u || (bf16x2 & 0x7f800000u) == 0x7f800000u;
}

}  // namespace dsv2

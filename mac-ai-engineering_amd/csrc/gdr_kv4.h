// The format of a paged cache of keys and values in 4 bits, shared by the kernels that fill, read and attend over it.
//
// A group of 32 channels of one key or value is 32 codes of 4 bits (E2M1: a sign and a magnitude of 0, 0.5, 1, 1.5, 2, 3,
// 4 or 6) and one power of two 2^(byte - 127), the OCP microscaling format whose conversions gfx950 has as instructions
// (v_cvt_scalef32_pk_bf16_fp4 and its inverse: exact, 0.5 instructions a value).  The scale is the smallest with which
// the group's largest magnitude is at most 7: up to there the 6 it rounds to is no further off than a value between 4
// and 6 may be (over N(0, 1) groups the error is 0.112 of the values' norm; 0.115 with largest magnitudes up to 6 or 8).
// A group that holds an infinity or a NaN has the byte 255 and reads as NaN.
//
// cache [pages, 2 (keys, values), heads, bytes a page-head]; a page-head is its blocks of 16 tokens, each 8 D bytes of
// codes and D / 2 of scales, ordered as a wave of the attention kernel loads them: lane l = 16 h + m of it takes
//   keys    token m, 32 channels of group 4 c + h: 16 bytes at c * 1024 + 16 l        ([D / 32 groups][16 tokens][16 B])
//   values  tokens 4 h .. 4 h + 3, channels 128 c + 8 m .. + 7: 16 bytes at c * 1024 + 16 l
//                                                                 ([D / 128][4 quads][16][4 tokens][4 B])
// for c < D / 128 (heads of 64: one load of 8 bytes, half a group of a key, 4 channels of a value), whole kilobytes
// without a gap, and a token's codes are still whole words, so appending one token writes no byte of another.
// Scales: keys [D / 32 groups][16 tokens], values [4 quads][D / 32 groups][4 tokens].
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gdr {

constexpr int KV_SUB = 16;                                                     // tokens of a block
__host__ __device__ constexpr int kv_sub_bytes(int D) { return 17 * D / 2; }   // one head's keys or values of a block
__host__ __device__ constexpr int64_t kv_page_bytes(int page, int D) { return (int64_t)(page / KV_SUB) * kv_sub_bytes(D); }

// Byte offsets in a block, for token t < 16 and channel ch (a multiple of 8; of 4 for values of heads of 64).
__device__ __forceinline__ int kv_key_code(int t, int ch) { return (ch >> 5) * 256 + t * 16 + ((ch & 31) >> 1); }
__device__ __forceinline__ int kv_key_scale(int D, int t, int group) { return 8 * D + group * 16 + t; }
__device__ __forceinline__ int kv_value_code(int D, int t, int ch) {
  const int W = D < 128 ? D : 128, wb = W / 32;                                // bytes of a run of W / 16 channels
  const int c = ch / W, m = (ch % W) / (2 * wb);
  return c * 8 * W + (t >> 2) * 64 * wb + m * 4 * wb + (t & 3) * wb;
}
__device__ __forceinline__ int kv_value_scale(int D, int t, int group) {
  return 8 * D + (t >> 2) * (D / 8) + group * 4 + (t & 3);
}

// The scale byte of a group whose largest magnitude has the float bits `top` (the sign cleared).
__device__ __forceinline__ unsigned kv_scale_byte(unsigned top) {
  const int e = (int)((top + 0x1FFFFFu) >> 23) - 2;
  return top >= 0x7F800000u ? 255u : (unsigned)min(max(e, 1), 252);
}
__device__ __forceinline__ float kv_scale(unsigned byte) { return __uint_as_float(byte << 23); }

// 8 values as 8 codes, value 2 i in the low half of byte i: rounded to nearest, ties to even, at most 6 in magnitude.
__device__ __forceinline__ unsigned kv_encode8(const float (&x)[8], float scale) {
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// Byte SEL of a word of codes as two bf16 values (exact: 2 bits of mantissa), the first in the low half.
template <int SEL>
__device__ __forceinline__ unsigned kv_decode2(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}

}  // namespace gdr

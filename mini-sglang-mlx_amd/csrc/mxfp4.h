// The format of a K/V pool in 4 bits, and the conversions both ways.
//
// A slot holds, for every kv head, D / 2 bytes of K and behind them D / 2 of V (the codes), and in a tensor of its own
// D / 32 bytes for K and D / 32 for V: one to each block of 32 dims.  A code is a 4-bit float (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6
// and a sign); dim 2 i is the low half of byte i, dim 2 i + 1 the high one.  A block byte b multiplies its block by 2^(b - 127).
// K and V of a head side by side are one line of 128 bytes (two at head_dim 256), which one wave reads whole.
//
// The block byte is the smallest with which nothing of the block lies beyond 6 (the largest code), so that no value is cut off: at most
// half a step of the code below is lost, 1/6 of a value above 4 and no more than 1/2 of the block's unit below 1.  It is held to
// [2, 252]: every value that a code can stand for is then a normal number in bf16 and in fp32, and what is finite stays finite.
// K or V that are not finite leave 255 in the block bytes of K, and zeros elsewhere: a score with such a key is NaN, and so is the
// result of who sees the key, while V, which meets a weight of zero where the mask hides the key, is always finite.
#pragma once
#include "msgl_device.h"

namespace msgl {

constexpr int kMxBlock = 32;
constexpr int kMxLeast = 2, kMxMost = 252;  // block bytes
constexpr int kMxNotFinite = 255;           // in K's

// The block byte for values up to the one with these bits (finite, not negative): with it m 2^e, 1 <= m < 2, the unit is 2^(e - 2) if 4 m <= 6, else 2^(e - 1).
__device__ __forceinline__ int mx_block_byte(uint32_t bits) {
  return min(max((int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0), kMxLeast), kMxMost);
}

// Eight values as codes, the first in the lowest 4 bits: divided by the block's unit (exact: of the factor the conversion takes the
// exponent), nearest, halfway to the even code.
__device__ __forceinline__ uint32_t mx_codes8(const float (&x)[8], int byte) {
  const float unit = __builtin_bit_cast(float, (uint32_t)byte << 23);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], unit, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], unit, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], unit, 3);
}

// Codes 2 B and 2 B + 1 of a word as bf16 or, with F16, IEEE half, times 2^(exponent of `scale`): of `scale` the conversion looks at
// the exponent alone, and 255 there gives NaN.  Exact in bf16, and in half where that reaches.
template <bool F16, int B>
__device__ __forceinline__ uint32_t mx_values2(uint32_t word, float scale) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, B));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, B));
}
template <bool F16>
__device__ __forceinline__ u32x4_t mx_values8(uint32_t word, float scale) {
  return u32x4_t{mx_values2<F16, 0>(word, scale), mx_values2<F16, 1>(word, scale), mx_values2<F16, 2>(word, scale),
                 mx_values2<F16, 3>(word, scale)};
}
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

}  // namespace msgl

// Rows in 4 bits: blocks of 32 elements, each a sign, two exponent and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6), two to
// a byte with the first in the low half, and a power of two for each block as a biased exponent byte (255: not finite).  The
// format is the OCP microscaling one that gfx950 converts in hardware, two elements an instruction, the power included.
#pragma once

#include <type_traits>

#include "biops_common.h"

namespace biops {

constexpr int kFp4Block = 32;

// Exponents of a block, biased: such that its values are normal numbers of the rows' type, or multiples of fp16's smallest
// one, so that what 4 bits hold is exact in 16.
template <typename T>
struct Fp4Range {
  static constexpr bool kHalf = std::is_same<T, f16_t>::value;
  static constexpr int kLow = 127 + (kHalf ? -23 : -125), kHigh = 127 + (kHalf ? 13 : 125);
};

// Elements 2 I and 2 I + 1 of the eight in a word of a block times its power of two (a float of the exponent byte in its place), in T.
template <typename T, int I>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t word, float power) {
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, power, I));
  else
    return __builtin_bit_cast(uint32_t, (f16x2_t)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, power, I));
}
// All eight.
template <typename T>
__device__ __forceinline__ u32x4_t fp4_values(uint32_t word, float power) {
  return u32x4_t{fp4_pair<T, 0>(word, power), fp4_pair<T, 1>(word, power), fp4_pair<T, 2>(word, power), fp4_pair<T, 3>(word, power)};
}

// The biased exponent of a block whose largest magnitude has the float bits `top`: the smallest power of two of which every
// value is at most 7 (the nearest level is then at most 1 away), 255 where one is not finite.
template <typename T>
__device__ __forceinline__ int fp4_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  const int e = (int)(top >> 23) - ((top & 0x7fffffu) <= 0x600000u ? 2 : 1);
  return e < Fp4Range<T>::kLow ? Fp4Range<T>::kLow : (e > Fp4Range<T>::kHigh ? Fp4Range<T>::kHigh : e);
}

// Eight elements in 4 bits: to the nearest level, to the even code where two are as near, past 6 to 6; zeros in a block that
// is not finite.
__device__ __forceinline__ uint32_t fp4_pack(const float (&x)[8], int exponent) {
  if (exponent == 255) return 0u;
  const float power = __uint_as_float((uint32_t)exponent << 23);
  uint32_t v = 0u;
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[0], x[1], power, 0);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[2], x[3], power, 1);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[4], x[5], power, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[6], x[7], power, 3);
}

}  // namespace biops

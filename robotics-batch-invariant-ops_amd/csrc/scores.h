// What the paged and the windowed attention share about scores: s_j = scale q.k_j, weights 2^(c (q.k_j - max)),
// c = |scale| log2 e, with the sign of a negative scale in the queries.
#pragma once

#include <cfloat>

#include "rowops.h"

namespace biops {

// c for the kernels, finite and not 0: masked scores are -inf, and c * -inf has to stay that.  A scale of 0 is c = 1 over
// queries of zeros (`zero`), so that weights are equal however large the products would be.
inline float score_scale(float scale, int* negate, int* zero) {
  const float c = (scale < 0.f ? -scale : scale) * kLog2e;
  *negate = scale < 0.f;
  *zero = c == 0.f;
  return c == 0.f ? 1.f : (c < FLT_MAX ? c : FLT_MAX);
}

// Exponent bits of an element: all of them are set where it is not finite.
template <typename T>
__host__ __device__ constexpr uint32_t score_inf() {
  return Num<T>::kBytes == 4 ? 0x7f800000u : (std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u);
}

// 0 * x of packed elements: 0, and NaN where x is not finite.
template <typename T>
__device__ __forceinline__ u32x4_t times_zero(u32x4_t v) {
  constexpr uint32_t inf = score_inf<T>(), nan = inf | inf >> 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Num<T>::kBytes == 4) v[i] = (v[i] & inf) == inf ? nan : 0u;
    else v[i] = ((v[i] & inf) == inf ? nan : 0u) | ((v[i] & inf << 16) == inf << 16 ? nan << 16 : 0u);
  }
  return v;
}

// Queries as the kernels multiply them.
template <typename T>
__device__ __forceinline__ u32x4_t score_query(u32x4_t v, int negate, int zero) {
  if (negate) v ^= Num<T>::kBytes == 2 ? 0x80008000u : 0x80000000u;
  return zero ? times_zero<T>(v) : v;
}

}  // namespace biops

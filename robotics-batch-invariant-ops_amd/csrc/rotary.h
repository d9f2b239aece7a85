// The rotation of rotary positions: what rotary.hip and cache_append.hip share.
#pragma once

#include "biops_common.h"

namespace biops {

constexpr int kRotaryPairs = 128;  // most pairs (a head size of 256 rotated whole)

struct RotaryTensor {
  const char* x;
  char* y;
  int64_t xB, xT, xH, yB, yT, yH;  // byte strides: batch, token, head
};

template <typename T>
__device__ __forceinline__ void unpack(const u32x4_t& v, float (&x)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Num<T>::from_bits(v[i] & 0xffffu);
      x[2 * i + 1] = Num<T>::from_bits(v[i] >> 16);
    }
  }
}
template <typename T>
__device__ __forceinline__ u32x4_t pack(const float (&x)[16 / sizeof(T)]) {
  u32x4_t v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(x[i]);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f32x2_to_f16x2_bits(x[2 * i], x[2 * i + 1]);
  }
  return v;
}
__device__ __forceinline__ void store_16(void* p, const u32x4_t& v) { *reinterpret_cast<u32x4_any_t*>(p) = v; }
// (PAST: past the caches)
template <bool PAST>
__device__ __forceinline__ void put_16(void* p, const u32x4_t& v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any_t*>(p));
  else store_16(p, v);
}

__device__ __forceinline__ void turn(float& x0, float& x1, float c, float s) {
  const float y0 = __builtin_fmaf(x0, c, -(x1 * s)), y1 = __builtin_fmaf(x1, c, x0 * s);
  x0 = y0;
  x1 = y1;
}

// Cosine and sine of the angle of the position at `at` (pos_type 0 int64, 1 int32, 2 float32), `turns` a position, in turns.
__device__ __forceinline__ void rotary_angle(const void* pos, int pos_type, int64_t at, double turns, float& c, float& s) {
  double p;
  if (pos_type == 0) p = (double)reinterpret_cast<const int64_t*>(pos)[at];
  else if (pos_type == 1) p = (double)reinterpret_cast<const int32_t*>(pos)[at];
  else p = (double)reinterpret_cast<const float*>(pos)[at];
  const double r = p * turns;
  sincospif(2.f * (float)(r - rint(r)), &s, &c);
}

// Pieces of a head of d elements: VEC pairs (both halves) or VEC / 2 neighbouring pairs, then what is copied.
template <typename T>
__device__ __forceinline__ int rotary_pieces(int S, int neighbours) {
  constexpr int VEC = 16 / sizeof(T);
  return neighbours ? (2 * S + VEC - 1) / VEC : (S + VEC - 1) / VEC;
}
// Piece c of a head from src to dst, np of them rotated; cs: S cosines, and the sines SP places behind them.
template <typename T, bool PAST = false>
__device__ __forceinline__ void rotary_piece(int c, int np, const T* src, T* dst, const float* cs, int S, int SP, int d, int neighbours) {
  constexpr int VEC = 16 / sizeof(T);
  if (c >= np) {  // copied
    const int e0 = 2 * S + (c - np) * VEC;
    if (e0 + VEC <= d) put_16<PAST>(dst + e0, load_16(src + e0));
    else
      for (int e = e0; e < d; ++e) dst[e] = src[e];
  } else if (neighbours) {
    const int e0 = c * VEC;
    if (e0 + VEC <= 2 * S) {
      float v[VEC];
      unpack<T>(load_16(src + e0), v);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) turn(v[2 * i], v[2 * i + 1], cs[e0 / 2 + i], cs[SP + e0 / 2 + i]);
      put_16<PAST>(dst + e0, pack<T>(v));
    } else {
      for (int e = e0; e < 2 * S; e += 2) {
        float v0 = Num<T>::load(src + e), v1 = Num<T>::load(src + e + 1);
        turn(v0, v1, cs[e / 2], cs[SP + e / 2]);
        Num<T>::store(dst + e, v0);
        Num<T>::store(dst + e + 1, v1);
      }
    }
  } else {
    const int e0 = c * VEC;
    if (e0 + VEC <= S) {
      float v0[VEC], v1[VEC];
      unpack<T>(load_16(src + e0), v0);
      unpack<T>(load_16(src + S + e0), v1);
#pragma unroll
      for (int i = 0; i < VEC; ++i) turn(v0[i], v1[i], cs[e0 + i], cs[SP + e0 + i]);
      put_16<PAST>(dst + e0, pack<T>(v0));
      put_16<PAST>(dst + S + e0, pack<T>(v1));
    } else {
      for (int e = e0; e < S; ++e) {
        float v0 = Num<T>::load(src + e), v1 = Num<T>::load(src + S + e);
        turn(v0, v1, cs[e], cs[SP + e]);
        Num<T>::store(dst + e, v0);
        Num<T>::store(dst + S + e, v1);
      }
    }
  }
}

}  // namespace biops

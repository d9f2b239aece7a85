// Rotary positions with several axes (time, height, width, ...) for queries and keys in one launch.
//
// Pair i of a head's S rotated pairs belongs to axis a(i) and turns by t = p * f_i, p the token's
// position on that axis: (x0, x1) -> (x0 cos t - x1 sin t, x1 cos t + x0 sin t).  Elements behind the
// 2 S rotated ones are copied.  The gradient is the same map with t negated.
//
// Far positions need more than 32 bits: p f_i / 2 pi (in turns) is formed in 64 bits, its whole turns
// are taken off, and only the rest in [-1/2, 1/2] goes to the 32-bit sine and cosine.  Rotation is in 32
// bits with one rounding to the tensor's type at the end.
//
// What bounds it is memory (each element read and written once).  A workgroup takes a few tokens: it
// computes their S cosines and sines once into LDS, where all heads of queries and keys find them, and
// then moves 16-byte pieces.
//
// The video case (32768 tokens, 16 + 4 heads of 128 in bf16, 336 MB): 66.5 us, 5.05 TB/s, the rate of a plain
// copy.  4100 tokens of 16 + 16 float32 heads of 72: 17.4 us (a copy 15).  16 tokens: 3.5 us, a launch.
// (Stores past the caches take 3 to 25 % less by themselves, and nothing off the rotation and its reader together.)
#include "biops_common.h"

namespace biops {

constexpr int kRotaryPairs = 128;  // most pairs (a head size of 256 rotated whole)

struct RotaryTensor {
  const char* x;
  char* y;
  int64_t xB, xT, xH, yB, yT, yH;  // byte strides: batch, token, head
};

struct RotaryArgs {
  double turns[kRotaryPairs];  // f_i / 2 pi
  uint8_t axis[kRotaryPairs];
  RotaryTensor t[2];           // queries, keys
  const void* pos;
  int64_t pA, pB, pT;          // element strides of the positions: axis, batch, token
  int64_t tokens, per_batch;   // all tokens, tokens of one batch entry
  int heads[2];
  int d, pairs, group;         // group: tokens per workgroup
  int pos_type;                // 0 int64, 1 int32, 2 float32
  int neighbours;              // pairs (2i, 2i + 1) instead of (i, i + S)
  float sign;
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

__device__ __forceinline__ void turn(float& x0, float& x1, float c, float s) {
  const float y0 = __builtin_fmaf(x0, c, -(x1 * s)), y1 = __builtin_fmaf(x1, c, x0 * s);
  x0 = y0;
  x1 = y1;
}

template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  extern __shared__ __attribute__((aligned(16))) float table[];  // [token][cos, sin][pairs padded to 8]
  constexpr int E = sizeof(T), VEC = 16 / E;
  // the tables are indexed per lane: read in the kernel's argument segment (a copy would go to scratch)
  const auto* args = (const __attribute__((address_space(4))) RotaryArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  const int tid = threadIdx.x;
  const int S = a.pairs, SP = (S + 7) & ~7;
  const int heads = a.heads[0] + a.heads[1];
  // pieces of a head: VEC pairs (both halves) or VEC / 2 neighbouring pairs, then what is copied
  const int np = a.neighbours ? (2 * S + VEC - 1) / VEC : (S + VEC - 1) / VEC;
  const int units = np + (a.d - 2 * S + VEC - 1) / VEC;
  for (int64_t t0 = (int64_t)blockIdx.x * a.group; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.group) {
    const int n = a.tokens - t0 < a.group ? (int)(a.tokens - t0) : a.group;
    for (int i = tid; i < n * S; i += 256) {
      const int tok = i / S, j = i - tok * S;
      const int64_t t = t0 + tok, b = t / a.per_batch;
      const int64_t at = args->axis[j] * a.pA + b * a.pB + (t - b * a.per_batch) * a.pT;
      double p;
      if (a.pos_type == 0) p = (double)reinterpret_cast<const int64_t*>(a.pos)[at];
      else if (a.pos_type == 1) p = (double)reinterpret_cast<const int32_t*>(a.pos)[at];
      else p = (double)reinterpret_cast<const float*>(a.pos)[at];
      const double r = p * args->turns[j];
      float s, c;
      sincospif(2.f * (float)(r - rint(r)), &s, &c);
      table[tok * 2 * SP + j] = c;
      table[tok * 2 * SP + SP + j] = s * a.sign;
    }
    __syncthreads();
    for (int u = tid; u < n * heads * units; u += 256) {
      const int c = u % units, th = u / units;
      int h = th % heads;
      const int tok = th / heads;
      const int64_t t = t0 + tok, b = t / a.per_batch, tb = t - b * a.per_batch;
      const int which = h >= a.heads[0];
      const RotaryTensor& x = a.t[which];
      if (which) h -= a.heads[0];
      const T* src = reinterpret_cast<const T*>(x.x + b * x.xB + tb * x.xT + h * x.xH);
      T* dst = reinterpret_cast<T*>(x.y + b * x.yB + tb * x.yT + h * x.yH);
      const float* cs = table + tok * 2 * SP;
      if (c >= np) {  // copied
        const int e0 = 2 * S + (c - np) * VEC;
        if (e0 + VEC <= a.d) store_16(dst + e0, load_16(src + e0));
        else
          for (int e = e0; e < a.d; ++e) dst[e] = src[e];
      } else if (a.neighbours) {
        const int e0 = c * VEC;
        if (e0 + VEC <= 2 * S) {
          float v[VEC];
          unpack<T>(load_16(src + e0), v);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) turn(v[2 * i], v[2 * i + 1], cs[e0 / 2 + i], cs[SP + e0 / 2 + i]);
          store_16(dst + e0, pack<T>(v));
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
          store_16(dst + e0, pack<T>(v0));
          store_16(dst + S + e0, pack<T>(v1));
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
    __syncthreads();
  }
}

static int rotary_launch(int dtype, const RotaryArgs& a, hipStream_t s) {
  const int64_t groups = cdiv(a.tokens, a.group);
  const unsigned blocks = (unsigned)(groups < (1 << 20) ? groups : (1 << 20));
  const unsigned lds = (unsigned)(a.group * 2 * ((a.pairs + 7) & ~7) * sizeof(float));
  BIOPS_DISPATCH_FLOAT(dtype, hipLaunchKernelGGL((rotary_kernel<T>), dim3(blocks), dim3(256), lds, s, a));
  return check_launch("rotary_kernel");
}

}  // namespace biops

using namespace biops;

extern "C" int biops_rotary(int dtype, int64_t batch, int64_t tokens, int64_t hq, int64_t hk, int64_t d,
                            const void* q, int64_t sqB, int64_t sqT, int64_t sqH, void* oq, int64_t soqB, int64_t soqT,
                            int64_t soqH, const void* k, int64_t skB, int64_t skT, int64_t skH, void* ok, int64_t sokB,
                            int64_t sokT, int64_t sokH, const void* positions, int pos_type, int64_t spA, int64_t spB,
                            int64_t spT, int64_t pairs, const double* turns, const uint8_t* axis, int neighbours,
                            int inverse, void* stream) {
  const int elt = is_float_dtype(dtype) ? dtype_bytes(dtype) : 0;
  if (elt == 0) return fail(BIOPS_ERR_DTYPE, "biops_rotary: unsupported dtype %d", dtype);
  if (batch < 0 || tokens < 0 || hq < 0 || hk < 0 || hq + hk > 65536 || d < 0 || d > (1 << 20))
    return fail(BIOPS_ERR_ARG, "biops_rotary: bad sizes");
  if ((hq + hk) * d > (INT64_C(1) << 26)) return fail(BIOPS_ERR_ARG, "biops_rotary: tokens of more than 2^26 elements");
  if (pairs < 0 || pairs > kRotaryPairs || 2 * pairs > d)
    return fail(BIOPS_ERR_ARG, "biops_rotary: %lld pairs (at most %d, and half the head size)", (long long)pairs, kRotaryPairs);
  if (pos_type < 0 || pos_type > 2) return fail(BIOPS_ERR_DTYPE, "biops_rotary: bad position type %d", pos_type);
  if (batch == 0 || tokens == 0 || hq + hk == 0 || d == 0) return BIOPS_OK;
  if (tokens > (INT64_C(1) << 40) / batch) return fail(BIOPS_ERR_ARG, "biops_rotary: too many tokens");
  if ((hq > 0 && (!q || !oq)) || (hk > 0 && (!k || !ok)) || (pairs > 0 && (!positions || !turns || !axis)))
    return fail(BIOPS_ERR_ARG, "biops_rotary: null pointer");
  RotaryArgs a;
  for (int i = 0; i < kRotaryPairs; ++i) {
    a.turns[i] = i < pairs ? turns[i] : 0.0;
    a.axis[i] = i < pairs ? axis[i] : 0;
  }
  a.t[0] = RotaryTensor{static_cast<const char*>(q), static_cast<char*>(oq), elt * sqB, elt * sqT, elt * sqH,
                        elt * soqB, elt * soqT, elt * soqH};
  a.t[1] = RotaryTensor{static_cast<const char*>(k), static_cast<char*>(ok), elt * skB, elt * skT, elt * skH,
                        elt * sokB, elt * sokT, elt * sokH};
  a.pos = positions;
  a.pA = spA, a.pB = spB, a.pT = spT;
  a.tokens = batch * tokens, a.per_batch = tokens;
  a.heads[0] = (int)hq, a.heads[1] = (int)hk;
  a.d = (int)d, a.pairs = (int)pairs;
  a.pos_type = pos_type, a.neighbours = neighbours != 0;
  a.sign = inverse ? -1.f : 1.f;
  // Few tokens: one per workgroup spreads them over the chip.  Many: four fill its threads and share its start.
  // us (one / two / four / eight), 16 + 4 bf16 heads of 128: 16 tokens 3.5 / 4.1 / 4.5 / 6.3, 2048 6.9 / 6.8 / 7.1 / 8.8,
  // 4096 11.8 / 11.7 / 10.2 / 11.4, 32768 84 / 71 / 66 / 68; 16 + 16 float32 heads of 72: 2048 12 / 11 / 13 / 20,
  // 4096 17.8 / 17.9 / 16.9 / 23.
  a.group = a.tokens >= 4096 ? 4 : 1;
  return rotary_launch(dtype, a, static_cast<hipStream_t>(stream));
}

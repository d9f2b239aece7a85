// New keys and values on their way into a cache in pages: keys turned by their positions (queries too, into a tensor of their
// own), rows in the cache's type or in 4 bits (fp4.h), and rows in 4 bits read back as values.
//
// The rotation is that of rotary.hip and the rows go where paged_cache.hip puts them, bit for bit: row r's keys and values to
// slot slots[r], none where the slot is negative or past the cache (which the flag reports), and of rows that name one slot
// the last stays.  In 4 bits a key is rotated and rounded to its type first, so what is written is what rotation and write
// one after another would leave.
//
// Memory bounds it: each element read and written once, without the rotated keys' way out and back.  A workgroup takes one
// row, or several that share a search for rows behind them with the same slot; it computes the rows' cosines and sines into
// LDS, where all heads find them, and moves 16-byte pieces.  In 4 bits a lane has 8 elements of a block, four lanes share
// the block's power of two, and the rotation's partners are read a second time (from the caches) instead of exchanged.
#include "cache_slots.h"
#include "fp4.h"
#include "rotary.h"

namespace biops {

struct AppendArgs {
  double turns[kRotaryPairs];
  uint8_t axis[kRotaryPairs];
  const char *q, *k, *v;
  char *oq, *kc, *vc, *ks, *vs;
  int64_t qT, qH, oqT, oqH, kT, kH, vT, vH;                  // byte strides: row, head
  int64_t kcP, kcS, kcH, vcP, vcS, vcH;                      // page, slot, head
  int64_t ksP, ksS, ksH, vsP, vsS, vsH;
  const void *pos, *slots;
  int64_t pA, pT, slot_stride;                               // element strides
  int* flag;
  uint32_t total, page;                                      // slots of the cache, slots of a page
  int rows, hq, hk, d, dv, pairs, pos_type, neighbours, slots64;
};

typedef uint32_t u32_byte_t __attribute__((aligned(1)));

// Elements e0 .. e0 + 7 (e0 a multiple of 8) of a head after its rotation, rounded to T.
template <typename T>
__device__ __forceinline__ void rotated_eight(const T* src, int e0, const float* cs, int S, int SP, int neighbours, float (&y)[8]) {
  unpack<T>(load_16(src + e0), y);
  if (e0 >= 2 * S) return;
  if (neighbours) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e0 + 2 * i < 2 * S) turn(y[2 * i], y[2 * i + 1], cs[e0 / 2 + i], cs[SP + e0 / 2 + i]);
  } else if (S % 8 == 0) {
    const bool first = e0 < S;
    float x[8];
    unpack<T>(load_16(src + (first ? e0 + S : e0 - S)), x);
    const float* at = cs + (first ? e0 : e0 - S);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x0 = first ? y[i] : x[i], x1 = first ? x[i] : y[i];
      turn(x0, x1, at[i], at[SP + i]);
      y[i] = first ? x0 : x1;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i;
      if (e >= 2 * S) continue;
      const bool first = e < S;
      const int j = first ? e : e - S;
      float x0 = Num<T>::load(src + j), x1 = Num<T>::load(src + j + S);
      turn(x0, x1, cs[j], cs[SP + j]);
      y[i] = first ? x0 : x1;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = Num<T>::round(y[i]);
}

// Eight elements of a block (the next three lanes have the others, or those before) to `data`, its exponent to `exponents`.
template <typename T>
__device__ __forceinline__ void store_eight(const float (&y)[8], int e0, char* data, char* exponents, bool stays) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t x = __float_as_uint(y[i]) & 0x7fffffffu;
    top = x > top ? x : top;
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const uint32_t x = (uint32_t)__shfl_xor((int)top, o, 64);
    top = x > top ? x : top;
  }
  const int e = fp4_exponent<T>(top);
  if (!stays) return;
  *reinterpret_cast<u32_byte_t*>(data + (e0 >> 1)) = fp4_pack(y, e);
  if (e0 % kFp4Block == 0) exponents[e0 / kFp4Block] = (char)e;
}

// FOUR: the cache is in 4 bits (T: bf16 or fp16); G: rows of a workgroup.
template <typename T, bool FOUR, int G>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  extern __shared__ __attribute__((aligned(16))) float table[];  // [row][cos, sin][pairs padded to 8]
  __shared__ int64_t place[G];
  __shared__ int again[G];
  constexpr int E = sizeof(T), VEC = 16 / E;
  // the tables are indexed per lane: read in the kernel's argument segment (a copy would go to scratch)
  const auto* args = (const __attribute__((address_space(4))) AppendArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * G;
  const int n = a.rows - r0 < G ? a.rows - r0 : G;
  const int S = a.pairs, SP = (S + 7) & ~7;
  auto slot = [&](int r) -> int64_t {
    return a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[r * a.slot_stride]
                     : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[r * a.slot_stride];
  };
  int64_t first = -1;
  if (tid < n) first = slot(r0 + tid);
  for (int i = tid; i < n * S; i += 256) {
    const int r = i / S, j = i - r * S;
    float c, s;
    rotary_angle(a.pos, a.pos_type, args->axis[j] * a.pA + (r0 + r) * a.pT, args->turns[j], c, s);
    table[r * 2 * SP + j] = c;
    table[r * 2 * SP + SP + j] = s;
  }
  slots_that_stay<G>(slot, r0, a.rows, first, a.total, a.flag, place, again);

  // pieces: keys, values (in 4 bits a multiple of four each, so that a block's four lanes are together), queries
  const int np = rotary_pieces<T>(S, a.neighbours), whole = np + (a.d - 2 * S + VEC - 1) / VEC;
  const int kn = FOUR ? a.d / 8 : whole, vn = FOUR ? a.dv / 8 : (a.dv + VEC - 1) / VEC;
  const int keys = n * a.hk * kn, values = n * a.hk * vn, queries = n * a.hq * whole;
  for (int u = tid; u < keys + values + queries; u += 256) {
    if (u < keys) {
      const int c = u % kn, rh = u / kn, h = rh % a.hk, r = rh / a.hk;
      const T* src = reinterpret_cast<const T*>(a.k + (r0 + r) * a.kT + h * a.kH);
      const float* cs = table + r * 2 * SP;
      const bool stays = place[r] >= 0 && !again[r];
      const uint32_t s = stays ? (uint32_t)place[r] : 0u, page = s / a.page, at = s - page * a.page;
      char* const dst = a.kc + page * a.kcP + at * a.kcS + h * a.kcH;
      if constexpr (FOUR) {
        float y[8];
        rotated_eight<T>(src, 8 * c, cs, S, SP, a.neighbours, y);
        store_eight<T>(y, 8 * c, dst, a.ks + page * a.ksP + at * a.ksS + h * a.ksH, stays);
      } else if (stays) {
        rotary_piece<T>(c, np, src, reinterpret_cast<T*>(dst), cs, S, SP, a.d, a.neighbours);
      }
    } else if (u < keys + values) {
      const int x = u - keys;
      const int c = x % vn, rh = x / vn, h = rh % a.hk, r = rh / a.hk;
      const T* src = reinterpret_cast<const T*>(a.v + (r0 + r) * a.vT + h * a.vH);
      const bool stays = place[r] >= 0 && !again[r];
      const uint32_t s = stays ? (uint32_t)place[r] : 0u, page = s / a.page, at = s - page * a.page;
      char* const dst = a.vc + page * a.vcP + at * a.vcS + h * a.vcH;
      if constexpr (FOUR) {
        float y[8];
        unpack<T>(load_16(src + 8 * c), y);
        store_eight<T>(y, 8 * c, dst, a.vs + page * a.vsP + at * a.vsS + h * a.vsH, stays);
      } else if (stays) {
        T* const to = reinterpret_cast<T*>(dst);
        if (VEC * (c + 1) <= a.dv) store_16(to + VEC * c, load_16(src + VEC * c));
        else
          for (int e = VEC * c; e < a.dv; ++e) to[e] = src[e];
      }
    } else {
      const int x = u - keys - values;
      const int c = x % whole, rh = x / whole, h = rh % a.hq, r = rh / a.hq;
      rotary_piece<T>(c, np, reinterpret_cast<const T*>(a.q + (r0 + r) * a.qT + h * a.qH),
                      reinterpret_cast<T*>(a.oq + (r0 + r) * a.oqT + h * a.oqH), table + r * 2 * SP, S, SP, a.d, a.neighbours);
    }
  }
}

template <typename T, bool FOUR>
static int append_launch(const AppendArgs& a, hipStream_t s) {
  constexpr int kFew = 1024, kGroup = 4;
  const int group = a.rows <= kFew ? 1 : kGroup;
  const dim3 grid((unsigned)cdiv(a.rows, group));
  const unsigned lds = (unsigned)(group * 2 * ((a.pairs + 7) & ~7) * sizeof(float));
  if (group == 1) hipLaunchKernelGGL((append_kernel<T, FOUR, 1>), grid, dim3(256), lds, s, a);
  else hipLaunchKernelGGL((append_kernel<T, FOUR, kGroup>), grid, dim3(256), lds, s, a);
  return check_launch("append_kernel");
}

struct ReadArgs {
  const char *kc, *vc, *ks, *vs;
  char *ok, *ov;                                // [rows, heads, d], [rows, heads, dv]
  int64_t kcP, kcS, kcH, vcP, vcS, vcH;         // byte strides
  int64_t ksP, ksS, ksH, vsP, vsS, vsH;
  const void* slots;
  int64_t slot_stride;
  int* flag;
  uint32_t total, page;
  int64_t rows;
  int heads, d, dv, slots64;
};

// Eight elements a thread and step; pieces of a row are its heads' keys, then its heads' values.
template <typename T>
__global__ __launch_bounds__(256) void read4_kernel(ReadArgs a) {
  const int kn = a.heads * (a.d / 8), per_row = kn + a.heads * (a.dv / 8);
  const int64_t all = a.rows * per_row;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += (int64_t)gridDim.x * 256) {
    const int64_t r = u / per_row;
    int x = (int)(u - r * per_row);
    const bool value = x >= kn;
    if (value) x -= kn;
    const int width = value ? a.dv : a.d;
    const int h = x / (width / 8), e0 = 8 * (x - h * (width / 8));
    const int64_t s = a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[r * a.slot_stride]
                                : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[r * a.slot_stride];
    u32x4_t y = {0u, 0u, 0u, 0u};
    if (s >= 0 && s < (int64_t)a.total) {
      const uint32_t page = (uint32_t)s / a.page, at = (uint32_t)s - page * a.page;
      const char* data = value ? a.vc + page * a.vcP + at * a.vcS + h * a.vcH : a.kc + page * a.kcP + at * a.kcS + h * a.kcH;
      const char* exps = value ? a.vs + page * a.vsP + at * a.vsS + h * a.vsH : a.ks + page * a.ksP + at * a.ksS + h * a.ksH;
      const uint32_t e = (uint8_t)exps[e0 / kFp4Block];
      y = fp4_values<T>(*reinterpret_cast<const u32_byte_t*>(data + (e0 >> 1)), __uint_as_float(e << 23));
    } else if (s >= 0) {
      *a.flag = 1;
    }
    store_16((value ? a.ov : a.ok) + 2 * ((r * a.heads + h) * width + e0), y);
  }
}

}  // namespace biops

using namespace biops;

static int append_sizes(const char* what, int64_t rows, int64_t hq, int64_t hk, int64_t d, int64_t dv, int64_t pages, int64_t page_size) {
  if (rows < 0 || hq < 0 || hk < 0 || d < 0 || dv < 0 || pages < 0 || page_size < 0 || rows > (INT64_C(1) << 40))
    return fail(BIOPS_ERR_ARG, "%s: negative or huge size", what);
  if (page_size > 0 && pages > INT64_C(0x7fffffff) / page_size) return fail(BIOPS_ERR_ARG, "%s: a cache of more than 2^31 - 1 slots", what);
  if (hq > (1 << 20) || hk > (1 << 20) || d > (1 << 20) || dv > (1 << 20) || (hq + hk) * d + hk * dv > (1 << 22))
    return fail(BIOPS_ERR_ARG, "%s: rows of more than 2^22 elements", what);
  return BIOPS_OK;
}

extern "C" int biops_rotary_write(int dtype, int64_t rows, int64_t hq, int64_t hk, int64_t d, int64_t dv, const void* q,
                                  int64_t sqT, int64_t sqH, void* oq, int64_t soqT, int64_t soqH, const void* k, int64_t skT,
                                  int64_t skH, const void* v, int64_t svT, int64_t svH, void* kc, int64_t skcP, int64_t skcS,
                                  int64_t skcH, void* ks, int64_t sksP, int64_t sksS, int64_t sksH, void* vc, int64_t svcP,
                                  int64_t svcS, int64_t svcH, void* vs, int64_t svsP, int64_t svsS, int64_t svsH, int64_t pages,
                                  int64_t page_size, const void* slots, int slots64, int64_t slot_stride, const void* positions,
                                  int pos_type, int64_t spA, int64_t spT, int64_t pairs, const double* turns, const uint8_t* axis,
                                  int neighbours, int* flag, void* stream) {
  const int elt = is_float_dtype(dtype) ? dtype_bytes(dtype) : 0;
  const bool four = ks != nullptr || vs != nullptr;
  if (elt == 0 || (four && elt != 2)) return fail(BIOPS_ERR_DTYPE, "biops_rotary_write: unsupported dtype %d", dtype);
  if (const int rc = append_sizes("biops_rotary_write", rows, hq, hk, d, dv, pages, page_size)) return rc;
  if (pairs < 0 || pairs > kRotaryPairs || 2 * pairs > d)
    return fail(BIOPS_ERR_ARG, "biops_rotary_write: %lld pairs (at most %d, and half the head size)", (long long)pairs, kRotaryPairs);
  if (pos_type < 0 || pos_type > 2) return fail(BIOPS_ERR_DTYPE, "biops_rotary_write: bad position type %d", pos_type);
  if (four && (d % kFp4Block || dv % kFp4Block))
    return fail(BIOPS_ERR_ARG, "biops_rotary_write: head sizes in 4 bits are multiples of %d", kFp4Block);
  if (rows == 0 || (hq * d == 0 && hk * (d + dv) == 0)) return BIOPS_OK;
  if (!slots || !flag || (hq * d > 0 && (!q || !oq)) || (hk * d > 0 && !k) || (hk * dv > 0 && !v) ||
      (pairs > 0 && (!positions || !turns || !axis)))
    return fail(BIOPS_ERR_ARG, "biops_rotary_write: null pointer");
  if (pages * page_size > 0 && ((hk * d > 0 && (!kc || (four && !ks))) || (hk * dv > 0 && (!vc || (four && !vs)))))
    return fail(BIOPS_ERR_ARG, "biops_rotary_write: null cache");
  AppendArgs a;
  for (int i = 0; i < kRotaryPairs; ++i) {
    a.turns[i] = i < pairs ? turns[i] : 0.0;
    a.axis[i] = i < pairs ? axis[i] : 0;
  }
  const int64_t held = four ? 1 : elt;  // bytes of the caches' stride unit
  a.kc = static_cast<char*>(kc), a.vc = static_cast<char*>(vc), a.ks = static_cast<char*>(ks), a.vs = static_cast<char*>(vs);
  a.qT = elt * sqT, a.qH = elt * sqH, a.oqT = elt * soqT, a.oqH = elt * soqH;
  a.kT = elt * skT, a.kH = elt * skH, a.vT = elt * svT, a.vH = elt * svH;
  a.kcP = held * skcP, a.kcS = held * skcS, a.kcH = held * skcH;
  a.vcP = held * svcP, a.vcS = held * svcS, a.vcH = held * svcH;
  a.ksP = sksP, a.ksS = sksS, a.ksH = sksH, a.vsP = svsP, a.vsS = svsS, a.vsH = svsH;
  a.pA = spA, a.pT = spT, a.slot_stride = slot_stride, a.flag = flag;
  a.total = (uint32_t)(pages * page_size), a.page = page_size > 0 ? (uint32_t)page_size : 1u;
  a.hq = (int)hq, a.hk = (int)hk, a.d = (int)d, a.dv = (int)dv, a.pairs = (int)pairs;
  a.pos_type = pos_type, a.neighbours = neighbours != 0, a.slots64 = slots64 != 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t r = 0; r < rows; r += kWriteRows) {
    a.rows = (int)(rows - r < kWriteRows ? rows - r : kWriteRows);
    a.q = static_cast<const char*>(q) + r * a.qT, a.oq = static_cast<char*>(oq) + r * a.oqT;
    a.k = static_cast<const char*>(k) + r * a.kT, a.v = static_cast<const char*>(v) + r * a.vT;
    a.pos = static_cast<const char*>(positions) + r * spT * (pos_type == 0 ? 8 : 4);
    a.slots = static_cast<const char*>(slots) + r * slot_stride * (slots64 ? 8 : 4);
    int rc;
    if (four) rc = dtype == BIOPS_F16 ? append_launch<f16_t, true>(a, s) : append_launch<bf16_t, true>(a, s);
    else if (dtype == BIOPS_F32) rc = append_launch<float, false>(a, s);
    else rc = dtype == BIOPS_F16 ? append_launch<f16_t, false>(a, s) : append_launch<bf16_t, false>(a, s);
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}

extern "C" int biops_paged_read_fp4(int dtype, int64_t rows, int64_t heads, int64_t d, int64_t dv, const void* kc, int64_t skcP,
                                    int64_t skcS, int64_t skcH, const void* ks, int64_t sksP, int64_t sksS, int64_t sksH,
                                    const void* vc, int64_t svcP, int64_t svcS, int64_t svcH, const void* vs, int64_t svsP,
                                    int64_t svsS, int64_t svsH, int64_t pages, int64_t page_size, const void* slots, int slots64,
                                    int64_t slot_stride, void* ok, void* ov, int* flag, void* stream) {
  if (dtype != BIOPS_F16 && dtype != BIOPS_BF16) return fail(BIOPS_ERR_DTYPE, "biops_paged_read_fp4: unsupported dtype %d", dtype);
  if (const int rc = append_sizes("biops_paged_read_fp4", rows, 0, heads, d, dv, pages, page_size)) return rc;
  if (d % kFp4Block || dv % kFp4Block) return fail(BIOPS_ERR_ARG, "biops_paged_read_fp4: head sizes are multiples of %d", kFp4Block);
  if (rows == 0 || heads * (d + dv) == 0) return BIOPS_OK;
  if (!slots || !flag || (d > 0 && !ok) || (dv > 0 && !ov)) return fail(BIOPS_ERR_ARG, "biops_paged_read_fp4: null pointer");
  if (pages * page_size > 0 && ((d > 0 && (!kc || !ks)) || (dv > 0 && (!vc || !vs))))
    return fail(BIOPS_ERR_ARG, "biops_paged_read_fp4: null cache");
  ReadArgs a;
  a.kc = static_cast<const char*>(kc), a.vc = static_cast<const char*>(vc);
  a.ks = static_cast<const char*>(ks), a.vs = static_cast<const char*>(vs);
  a.ok = static_cast<char*>(ok), a.ov = static_cast<char*>(ov);
  a.kcP = skcP, a.kcS = skcS, a.kcH = skcH, a.vcP = svcP, a.vcS = svcS, a.vcH = svcH;
  a.ksP = sksP, a.ksS = sksS, a.ksH = sksH, a.vsP = svsP, a.vsS = svsS, a.vsH = svsH;
  a.slots = slots, a.slot_stride = slot_stride, a.flag = flag, a.slots64 = slots64 != 0;
  a.total = (uint32_t)(pages * page_size), a.page = page_size > 0 ? (uint32_t)page_size : 1u;
  a.rows = rows, a.heads = (int)heads, a.d = (int)d, a.dv = (int)dv;
  const int64_t blocks = cdiv(rows * heads * ((d + dv) / 8), 256);
  const dim3 grid((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == BIOPS_F16) hipLaunchKernelGGL((read4_kernel<f16_t>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((read4_kernel<bf16_t>), grid, dim3(256), 0, s, a);
  return check_launch("read4_kernel");
}

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
//
// Up to 1024 rows a workgroup has one row and looks for rows behind it itself (48 rows of 16/4 heads of 128 4.7 us, which
// is a launch).  More rows are compared in a launch of their own, 16383 rows in 5 us and 32768 in 12, and then come in groups
// that share the arithmetic of addresses, with stores that go past the caches: 16383 rows of 16/4 heads of 96 in fp16 30 us,
// 5.0 TB/s of what has to move, where a copy of 1 GiB reaches 5.1 (10 us more with stores into the caches).  In 4 bits 32768
// rows of 4 heads of 128 take 18 us, 4.7 TB/s, and 36045 rows 22 us back, 4.2 TB/s.
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
  uint8_t* stays;                                            // [kStayParts][rows] whether no part of the later rows has its slot (null: to be found here)
  uint32_t total, page;                                      // slots of the cache, slots of a page
  int rows, hq, hk, d, dv, pairs, pos_type, neighbours, slots64;
};

typedef uint32_t u32_byte_t __attribute__((aligned(1)));
typedef u32x2_t u32x2_byte_t __attribute__((aligned(1)));

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

// 8 H elements of a block (4 / H lanes side by side have all of it) to `data`, the block's exponent to `exponents`.
template <typename T, int H>
__device__ __forceinline__ void store_part(const float (&y)[H][8], int e0, char* data, char* exponents, bool stays) {
  uint32_t top = 0u;
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = __float_as_uint(y[h][i]) & 0x7fffffffu;
      top = x > top ? x : top;
    }
#pragma unroll
  for (int o = 1; o < 4 / H; o <<= 1) {
    const uint32_t x = (uint32_t)__shfl_xor((int)top, o, 64);
    top = x > top ? x : top;
  }
  const int e = fp4_exponent<T>(top);
  if (!stays) return;
  if constexpr (H == 2) *reinterpret_cast<u32x2_byte_t*>(data + (e0 >> 1)) = u32x2_t{fp4_pack(y[0], e), fp4_pack(y[1], e)};
  else *reinterpret_cast<u32_byte_t*>(data + (e0 >> 1)) = fp4_pack(y[0], e);
  if (e0 % kFp4Block == 0) exponents[e0 / kFp4Block] = (char)e;
}

__device__ __forceinline__ int64_t slot_of(const AppendArgs& a, int r) {
  return a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[r * a.slot_stride]
                   : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[r * a.slot_stride];
}

// Which of many rows stay.  A workgroup has 256 rows and one part of the later ones: its slots go into a table in LDS, with the
// last of its rows that names each, and the later slots are looked up there where they lie between the smallest and the
// largest of its own.
constexpr int kStayRows = 65536;  // rows of a launch: the later ones are read by every workgroup
constexpr int kStayParts = 8;
__global__ __launch_bounds__(256) void stays_kernel(AppendArgs a) {
  constexpr int kPlaces = 1024;
  constexpr uint32_t kNone = 0xffffffffu;
  __shared__ uint32_t slots[kPlaces];
  __shared__ int last[kPlaces];
  __shared__ uint32_t lows[4], highs[4];
  const int tid = threadIdx.x, part = blockIdx.x % kStayParts, first = blockIdx.x / kStayParts * 256, r = first + tid;
  for (int i = tid; i < kPlaces; i += 256) {
    slots[i] = kNone;
    last[i] = -1;
  }
  const int64_t named = r < a.rows ? slot_of(a, r) : -1;
  const bool inside = named >= 0 && named < (int64_t)a.total;
  if (named >= (int64_t)a.total) *a.flag = 1;
  const uint32_t slot = (uint32_t)named;
  auto place = [](uint32_t s) { return (s * 2654435761u) >> 22; };
  uint32_t low = inside ? slot : kNone, high = inside ? slot : 0u;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t x = (uint32_t)__shfl_xor((int)low, o, 64), y = (uint32_t)__shfl_xor((int)high, o, 64);
    low = x < low ? x : low;
    high = y > high ? y : high;
  }
  if ((tid & 63) == 0) {
    lows[tid >> 6] = low;
    highs[tid >> 6] = high;
  }
  __syncthreads();
  uint32_t at = 0;
  if (inside) {
    for (at = place(slot);; at = (at + 1) % kPlaces) {  // (at most 256 of the 1024 places are taken)
      const uint32_t was = atomicCAS(&slots[at], kNone, slot);
      if (was == kNone || was == slot) break;
    }
    atomicMax(&last[at], r);
  }
  for (int i = 0; i < 4; ++i) {
    low = lows[i] < low ? lows[i] : low;
    high = highs[i] > high ? highs[i] : high;
  }
  __syncthreads();
  constexpr int kAhead = 8;
  auto row_at = [&](int i) { return i < a.rows ? i : a.rows - 1; };
  for (int base = first + 256 + 256 * kAhead * part; base < a.rows && low <= high; base += 256 * kAhead * kStayParts) {
    int64_t s[kAhead];
    if (a.slots64) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) s[j] = reinterpret_cast<const int64_t*>(a.slots)[row_at(base + 256 * j + tid) * a.slot_stride];
    } else {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) s[j] = reinterpret_cast<const int32_t*>(a.slots)[row_at(base + 256 * j + tid) * a.slot_stride];
    }
    uint32_t met[kAhead];  // (three of four places are free: most slots end here)
#pragma unroll
    for (int j = 0; j < kAhead; ++j) met[j] = slots[place((uint32_t)s[j])];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (met[j] == kNone || s[j] < (int64_t)low || s[j] > (int64_t)high || base + 256 * j + tid >= a.rows) continue;
      for (uint32_t i = place((uint32_t)s[j]); slots[i] != kNone; i = (i + 1) % kPlaces)
        if (slots[i] == (uint32_t)s[j]) {
          last[i] = a.rows;
          break;
        }
    }
  }
  __syncthreads();
  if (r < a.rows) a.stays[part * a.rows + r] = inside && last[at] == r;
}

// FOUR: the cache is in 4 bits (T: bf16 or fp16); G: rows of a workgroup; FEW: which rows stay is found here.
template <typename T, bool FOUR, int G, bool FEW>
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
  int64_t first = -1;
  if (tid < n) first = slot_of(a, r0 + tid);
  bool stays = true;
  if constexpr (!FEW) {
    static_assert(kStayParts * G <= 256, "a thread for each part of a row");
    if (tid < kStayParts * n) stays = a.stays[(tid / n) * a.rows + r0 + tid % n] != 0;
    if (tid < G) {
      place[tid] = first;
      again[tid] = 0;
    }
    __syncthreads();
    if (!stays) again[tid % n] = 1;
  }
  for (int i = tid; i < n * S; i += 256) {
    const int r = i / S, j = i - r * S;
    float c, s;
    rotary_angle(a.pos, a.pos_type, args->axis[j] * a.pA + (r0 + r) * a.pT, args->turns[j], c, s);
    table[r * 2 * SP + j] = c;
    table[r * 2 * SP + SP + j] = s;
  }
  if constexpr (FEW) slots_that_stay<G>([&](int r) { return slot_of(a, r); }, r0, a.rows, first, a.total, a.flag, place, again);
  else __syncthreads();

  // pieces: keys, values (in 4 bits quarters of blocks, or halves where there are many rows; a block's lanes are together), queries
  const int np = rotary_pieces<T>(S, a.neighbours), whole = np + (a.d - 2 * S + VEC - 1) / VEC;
  constexpr int H = FEW ? 1 : 2;
  const int kn = FOUR ? a.d / (8 * H) : whole, vn = FOUR ? a.dv / (8 * H) : (a.dv + VEC - 1) / VEC;
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
        float y[H][8];
#pragma unroll
        for (int i = 0; i < H; ++i) rotated_eight<T>(src, 8 * (H * c + i), cs, S, SP, a.neighbours, y[i]);
        store_part<T, H>(y, 8 * H * c, dst, a.ks + page * a.ksP + at * a.ksS + h * a.ksH, stays);
      } else if (stays) {
        rotary_piece<T, !FEW>(c, np, src, reinterpret_cast<T*>(dst), cs, S, SP, a.d, a.neighbours);
      }
    } else if (u < keys + values) {
      const int x = u - keys;
      const int c = x % vn, rh = x / vn, h = rh % a.hk, r = rh / a.hk;
      const T* src = reinterpret_cast<const T*>(a.v + (r0 + r) * a.vT + h * a.vH);
      const bool stays = place[r] >= 0 && !again[r];
      const uint32_t s = stays ? (uint32_t)place[r] : 0u, page = s / a.page, at = s - page * a.page;
      char* const dst = a.vc + page * a.vcP + at * a.vcS + h * a.vcH;
      if constexpr (FOUR) {
        float y[H][8];
#pragma unroll
        for (int i = 0; i < H; ++i) unpack<T>(load_16(src + 8 * (H * c + i)), y[i]);
        store_part<T, H>(y, 8 * H * c, dst, a.vs + page * a.vsP + at * a.vsS + h * a.vsH, stays);
      } else if (stays) {
        T* const to = reinterpret_cast<T*>(dst);
        if (VEC * (c + 1) <= a.dv) put_16<!FEW>(to + VEC * c, load_16(src + VEC * c));
        else
          for (int e = VEC * c; e < a.dv; ++e) to[e] = src[e];
      }
    } else {
      const int x = u - keys - values;
      const int c = x % whole, rh = x / whole, h = rh % a.hq, r = rh / a.hq;
      rotary_piece<T, !FEW>(c, np, reinterpret_cast<const T*>(a.q + (r0 + r) * a.qT + h * a.qH),
                      reinterpret_cast<T*>(a.oq + (r0 + r) * a.oqT + h * a.oqH), table + r * 2 * SP, S, SP, a.d, a.neighbours);
    }
  }
}

constexpr int kStayFew = 1024;  // rows up to which each workgroup looks for later rows itself

template <typename T, bool FOUR>
static int append_launch(const AppendArgs& a, hipStream_t s) {
  constexpr int kGroup = FOUR ? 16 : 4;
  const unsigned table = (unsigned)(2 * ((a.pairs + 7) & ~7) * sizeof(float));
  if (a.stays == nullptr) {
    hipLaunchKernelGGL((append_kernel<T, FOUR, 1, true>), dim3((unsigned)a.rows), dim3(256), table, s, a);
    return check_launch("append_kernel");
  }
  hipLaunchKernelGGL(stays_kernel, dim3((unsigned)(cdiv(a.rows, 256) * kStayParts)), dim3(256), 0, s, a);
  if (const int rc = check_launch("stays_kernel")) return rc;
  hipLaunchKernelGGL((append_kernel<T, FOUR, kGroup, false>), dim3((unsigned)cdiv(a.rows, kGroup)), dim3(256), kGroup * table, s, a);
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

// Eight elements a piece; pieces of a row are its heads' keys, then its heads' values.  A thread has AHEAD pieces, 256 apart,
// whose loads go out together.
template <typename T, int AHEAD>
__global__ __launch_bounds__(256) void read4_kernel(ReadArgs a) {
  // (a workgroup's first row in 64 bits, which all lanes share, the rest in 32: 36045 rows in 22 us, 25 with 64-bit divisions)
  const uint32_t kn = a.heads * (a.d / 8), per_row = kn + a.heads * (a.dv / 8);
  const uint64_t u0 = (uint64_t)blockIdx.x * (256 * AHEAD), r0 = u0 / per_row, all = (uint64_t)a.rows * per_row - u0;
  const uint32_t x0 = (uint32_t)(u0 - r0 * per_row);
  int64_t s[AHEAD];
  uint32_t h[AHEAD], e0[AHEAD];
  bool value[AHEAD];
  char* to[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const uint32_t u = threadIdx.x + 256 * i, rows = (x0 + u) / per_row;
    const int64_t r = (int64_t)(r0 + rows);
    uint32_t x = x0 + u - rows * per_row;
    value[i] = x >= kn;
    if (value[i]) x -= kn;
    const uint32_t width = value[i] ? a.dv : a.d;
    h[i] = x / (width / 8);
    e0[i] = 8 * (x - h[i] * (width / 8));
    to[i] = (value[i] ? a.ov : a.ok) + 2 * ((r * a.heads + h[i]) * (int64_t)width + e0[i]);
    s[i] = -1;
    if (u < all)
      s[i] = a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[r * a.slot_stride]
                       : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[r * a.slot_stride];
  }
  uint32_t codes[AHEAD], e[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    codes[i] = 0u;
    e[i] = 127u;
    if (s[i] >= 0 && s[i] < (int64_t)a.total) {
      const uint32_t page = (uint32_t)s[i] / a.page, at = (uint32_t)s[i] - page * a.page;
      const char* data = value[i] ? a.vc + page * a.vcP + at * a.vcS + h[i] * a.vcH : a.kc + page * a.kcP + at * a.kcS + h[i] * a.kcH;
      const char* exps = value[i] ? a.vs + page * a.vsP + at * a.vsS + h[i] * a.vsH : a.ks + page * a.ksP + at * a.ksS + h[i] * a.ksH;
      codes[i] = *reinterpret_cast<const u32_byte_t*>(data + (e0[i] >> 1));
      e[i] = (uint8_t)exps[e0[i] / kFp4Block];
    } else if (s[i] >= 0) {
      *a.flag = 1;
    }
  }
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (threadIdx.x + 256 * i < all) __builtin_nontemporal_store(fp4_values<T>(codes[i], __uint_as_float(e[i] << 23)), reinterpret_cast<u32x4_any_t*>(to[i]));
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

extern "C" int64_t biops_rotary_write_workspace_size(int64_t rows) {
  return rows <= kStayFew ? 0 : (rows < kStayRows ? rows : kStayRows) * kStayParts;
}

extern "C" int biops_rotary_write(int dtype, int64_t rows, int64_t hq, int64_t hk, int64_t d, int64_t dv, const void* q,
                                  int64_t sqT, int64_t sqH, void* oq, int64_t soqT, int64_t soqH, const void* k, int64_t skT,
                                  int64_t skH, const void* v, int64_t svT, int64_t svH, void* kc, int64_t skcP, int64_t skcS,
                                  int64_t skcH, void* ks, int64_t sksP, int64_t sksS, int64_t sksH, void* vc, int64_t svcP,
                                  int64_t svcS, int64_t svcH, void* vs, int64_t svsP, int64_t svsS, int64_t svsH, int64_t pages,
                                  int64_t page_size, const void* slots, int slots64, int64_t slot_stride, const void* positions,
                                  int pos_type, int64_t spA, int64_t spT, int64_t pairs, const double* turns, const uint8_t* axis,
                                  int neighbours, int* flag, void* workspace, int64_t workspace_bytes, void* stream) {
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
  const int64_t need = biops_rotary_write_workspace_size(rows);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(BIOPS_ERR_SIZE, "biops_rotary_write: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  if (need > 0 && reinterpret_cast<uintptr_t>(workspace) % 8) return fail(BIOPS_ERR_LAYOUT, "biops_rotary_write: workspace not 8-byte aligned");
  AppendArgs a;
  a.stays = need > 0 ? static_cast<uint8_t*>(workspace) : nullptr;
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
  for (int64_t r = 0; r < rows; r += kStayRows) {
    a.rows = (int)(rows - r < kStayRows ? rows - r : kStayRows);
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
  const int64_t pieces = rows * heads * ((d + dv) / 8);
  if (pieces > INT64_C(1) << 33) return fail(BIOPS_ERR_SIZE, "biops_paged_read_fp4: more than 2^36 elements");  // (2^31 threads)
  hipStream_t s = static_cast<hipStream_t>(stream);
  // One piece a thread spreads few of them over the card: 64 rows of 4 + 4 heads of 128 3.2 us, 4.5 with four.
  if (pieces < 256 * 1024) {
    const dim3 grid((unsigned)cdiv(pieces, 256));
    if (dtype == BIOPS_F16) hipLaunchKernelGGL((read4_kernel<f16_t, 1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((read4_kernel<bf16_t, 1>), grid, dim3(256), 0, s, a);
    return check_launch("read4_kernel");
  }
  const dim3 grid((unsigned)cdiv(pieces, 1024));
  if (dtype == BIOPS_F16) hipLaunchKernelGGL((read4_kernel<f16_t, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((read4_kernel<bf16_t, 4>), grid, dim3(256), 0, s, a);
  return check_launch("read4_kernel");
}

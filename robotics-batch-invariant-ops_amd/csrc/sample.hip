// The next token of each row of logits, from one uniform random number a row.
//
// With T the temperature, M the row's largest logit and w_i = exp((l_i - M) / T), tokens are ranked by their logits, equal
// ones by their index.  Of this order stays the beginning that every filter allows: the first k (top-k), those before which
// less than p of the weight of the first k has gone (top-p), those with w_i >= min-p.  The token is the first index whose
// running sum of the weights that stay is past u times all of them.
//
// Sums decide between neighbours, so they are exact: a weight is formed to 2^-33 of itself, by its own logit, the row's largest and
// T alone, and rounded once to a multiple of 2^-43; sums of those are integers, the same in any order.  A row's token depends on its
// own row only.
//
// A row's tokens are shared among `segs` workgroups, in five launches (few workgroups four, and one where a workgroup has a
// whole row):
//   top     a segment's largest and smallest logit;
//   bins    tokens by log2 of their weight in 2048 bins, each with its count and the sum of the places inside of it, which
//           bound its weight to 2^-11 (one 32-bit sum a token);
//   join    the bins over all segments, and those that a border can lie in;
//   sums    the weights in front of those bins, for every 512 tokens, and a list of the tokens inside of them;
//   finish  the list sorted, the borders in its running sums, the sums of 512 tokens completed, and the token.
// Calls without top-k and top-p go without bins and join.  Where the list is too long (thousands of tokens in a bin: equal
// logits, mostly) finish finds the borders by bisection over the row.
//
// 64 rows of 131072 in float32, 33.6 MB that are read three times (the second and third time mostly from the caches): 8, 15, 8, 19.5 and
// 11 us, bound by the arithmetic of 64-bit weights, in finish by steps that wait for one another.  (With 64-bit
// sums a bin, joined with the borders' list by the last workgroup of a launch, bins took 78 us and sums 73: fences make
// each of an XCD's writes visible to the others.)  One row of 32000: 3, 5, 10 and 7.5 us, each bound by a launch and a few
// reads that wait for one another.  64 rows of 131072 equal logits, by bisection, 1.1 ms.
#include "biops_common.h"

namespace biops {

constexpr int kSampleThreads = 512, kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048, kSampleInside = 32, kSampleList = 2048, kSampleSub = 512;
constexpr int kSampleMost = 1 << 20;           // tokens of a row: sums of that many weights fit 64 bits
constexpr int64_t kSampleAll = INT64_C(1) << 35;  // tokens of a call: a launch has less than 2^32 threads
constexpr int kSampleSubs = kSampleMost / kSampleSub;
constexpr int kSampleTable = 1024;
constexpr int kSampleSeg = 8192;               // most tokens of a segment: 14 bits of a bin's word count, 18 add up places
constexpr int kSamplePlace = 18;
constexpr uint32_t kSampleCounted = 128;       // tokens of a list that are compared with one another
constexpr uint32_t kNoIndex = 0xffffffffu;

struct SampleRow {    // what join finds, and what several workgroups would have to compute again
  double top, c;       // SampleWeight
  uint64_t lightest;   // the largest y that min-p lets pass: log2(1 / min-p)
  int64_t token;       // the answer where there is nothing to sample, -2 elsewhere
  uint32_t scale;
  int plo, phi, bk;    // bins of the border of top-p (of top-k, where there is no top-p), of top-k; -1: none
  uint32_t count;      // tokens in front of bin bk
  int unused;
};
struct SampleSeg {                // of a segment
  uint64_t top;                   // rank of the largest logit, 0 where nothing counts
  uint64_t all, before, weight;   // weight of all tokens, in front of bin plo, in front of bin bk
  float low;
};

struct SampleArgs {
  const char* logits;
  int64_t ld;                                   // bytes between rows
  const float *u, *temperature, *top_p, *min_p;  // of every row, or null
  const void* top_k;
  int64_t u_s, t_s, k_s, p_s, m_s;
  double t0, p0, m0;                            // of all rows
  int64_t k0;
  int64_t* out;
  int rows, vocab, segs, seg, subs, k64;        // seg: tokens of a workgroup, a multiple of kSampleSub * kSampleWaves
  int filters;                                  // there is a top-k or a top-p
  // workspace
  SampleRow* row;
  SampleSeg* part;                              // [rows][segs]
  uint64_t *sub, *list;                         // [rows][subs], [rows][kSampleList]
  uint32_t *bins, *listed;                      // [rows][segs][bins]; [rows] entries of the list
};

// Larger logits have larger keys; equal ones equal keys.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float float_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// A token's place in the order: larger ones first.
__device__ __forceinline__ uint64_t rank_of(float x, uint32_t index) { return (uint64_t)key_of(x) << 32 | (kNoIndex - index); }

// Eight logits from element i of a row on; -inf behind its end.
template <typename T>
__device__ __forceinline__ void eight_logits(const T* row, int i, int vocab, float (&x)[8]) {
  if (i + 8 <= vocab) {
    if constexpr (sizeof(T) == 4) {
      const u32x4_t a = load_16(row + i), b = load_16(row + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = __uint_as_float(a[j]);
        x[4 + j] = __uint_as_float(b[j]);
      }
    } else {
      const u32x4_t a = load_16(row + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = Num<T>::from_bits(a[j] & 0xffffu);
        x[2 * j + 1] = Num<T>::from_bits(a[j] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < vocab ? Num<T>::load(row + i + j) : -INFINITY;
  }
}

// Weights.  y = (M - l) log2 e / T in units of 2^-40 (at most 50, which is a weight of 0: logits of -inf and NaN have that);
// 2^-y from a table of 2^(-i / 1024) in 64 bits and 1 - 2^-r = t - t^2 / 2 + t^3 / 6, t = r ln 2 < 2^-10.5, in 32.  A weight is off by
// less than 2^-33 of itself (2^-33.23 at most, over all 2^30 remainders r), and a sum by at most that.
struct SampleWeight {
  double top, c;
  bool infinite;            // M is infinite: only logits of that count, alike
  uint32_t scale;           // places of 2^-26 octaves, times 2^32
  const double* table;
  __device__ __forceinline__ uint64_t octaves(float x) const {
    double y = fmin((top - (double)x) * c, 50.0);
    if (infinite) y = x == INFINITY ? 0.0 : 50.0;
    return (uint64_t)__double_as_longlong(y + 4096.0) & 0xfffffffffffffull;
  }
  // the place among all places of the bins, kSampleInside of each
  __device__ __forceinline__ uint32_t place(uint64_t y) const {
    const uint32_t b = __umulhi((uint32_t)(y >> 14), scale);
    return b < kSampleBins * kSampleInside ? b : kSampleBins * kSampleInside - 1;
  }
  __device__ __forceinline__ int bin(uint64_t y) const { return (int)(place(y) / kSampleInside); }
  // in units of 2^-43
  __device__ __forceinline__ uint64_t units(uint64_t y) const {
    const uint32_t hi = (uint32_t)(y >> 32), lo = (uint32_t)y;
    const double t = table[(hi & 255u) << 2 | lo >> 30];
    const float r = (float)(lo & 0x3fffffffu) * (float)(0.6931471805599453 / 1099511627776.0);  // ln 2 / 2^40
    const float off = r * __builtin_fmaf(r, __builtin_fmaf(r, 1.f / 6.f, -0.5f), 1.f);
    const double w = fma(-t, (double)off, t);
    const double sized = __hiloint2double(__double2hiint(w) + ((43 - (int)(hi >> 8)) << 20), __double2loint(w));
    return (uint64_t)__double_as_longlong(sized + 0x1p52) & 0xfffffffffffffull;  // to the nearest
  }
};
// The table, by the exponential's series for 2^(-i / 1024) = e^(-i ln 2 / 1024): 24 terms leave less than 2^-80.
struct SampleTable {
  double value[kSampleTable];
};
constexpr SampleTable make_table() {
  SampleTable t{};
  for (int i = 0; i < kSampleTable; ++i) {
    const double x = -0.6931471805599453 * i / kSampleTable;
    double sum = 1.0;
    for (int n = 24; n > 0; --n) sum = 1.0 + sum * x / n;
    t.value[i] = sum;
  }
  return t;
}
__device__ const SampleTable kTable = make_table();
// (__syncthreads before use)
__device__ __forceinline__ void fill_table(double* table) {
  static_assert(kSampleTable == 2 * kSampleThreads, "16 bytes a thread");
  reinterpret_cast<u32x4_t*>(table)[threadIdx.x] = reinterpret_cast<const u32x4_t*>(kTable.value)[threadIdx.x];
}

// v plus what the lanes that CTRL names have (row_shr or row_bcast; 0 where there is none, or the row of 16 is not in ROWS).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t plus_lane(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((uint64_t)hi << 32 | lo);
}
// Inclusive sums over the wavefront's lanes (all of them active): in rows of 16, then over the rows.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  v = plus_lane<0x111, 0xf>(v);  // row_shr:1
  v = plus_lane<0x112, 0xf>(v);
  v = plus_lane<0x114, 0xf>(v);
  v = plus_lane<0x118, 0xf>(v);
  v = plus_lane<0x142, 0xa>(v);  // row_bcast:15
  return plus_lane<0x143, 0xc>(v);  // row_bcast:31
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
  v = wave_scan64(v);
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}
// The sum in front of this thread and the sum of all, over the workgroup.
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t* waves, uint64_t& all) {
  const uint64_t scan = wave_scan64(v);
  __syncthreads();  // (the last sums have been read)
  if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = scan;
  __syncthreads();
  uint64_t before = scan - v;
  all = 0;
#pragma unroll
  for (int i = 0; i < kSampleWaves; ++i) {
    if (i < (int)(threadIdx.x >> 6)) before += waves[i];
    all += waves[i];
  }
  return before;
}
__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* waves) {
  v = wave_sum64(v);
  __syncthreads();  // (the last sums have been read)
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int i = 0; i < kSampleWaves; ++i) all += waves[i];
  return all;
}

__device__ __forceinline__ double row_value(const float* p, int64_t s, double all, int r) { return p ? (double)p[r * s] : all; }

// Shared memory of the steps; the table stays from one step to the next.
struct SampleTop {
  uint64_t tops[kSampleWaves];
  float lows[kSampleWaves];
};
struct SampleBins {
  uint32_t bins[kSampleBins];
};
struct SampleJoin {
  uint64_t waves[3][kSampleWaves];
  int found[3];
  uint64_t bounds[2];
  uint32_t count;
};
struct SampleSums {
  uint64_t item[kSampleList];
  uint32_t met, ready;
};
struct SampleFinish {
  uint64_t sub[kSampleSubs], item[kSampleList], other[kSampleThreads];
  int chosen;
  uint64_t left;
};
struct SampleShared {
  double table[kSampleTable];
  uint64_t waves[kSampleWaves];
  union {
    SampleTop top;
    SampleBins bins;
    SampleJoin join;
    SampleSums sums;
    SampleFinish finish;
  };
};

// --------------------------------------------------------------------------------- largest logits ----
template <typename T>
__device__ __forceinline__ void top_step(const SampleArgs& a, int seg, int r, SampleTop& sh) {
  const int tid = threadIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  const int end = (seg + 1) * a.seg < a.vocab ? (seg + 1) * a.seg : a.vocab;
  float best = -INFINITY, low = INFINITY;
  int at = -1;
  for (int i = seg * a.seg + 8 * tid; i < end; i += 8 * kSampleThreads) {
    float x[8];
    eight_logits<T>(row, i, a.vocab, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // (-inf and NaN do not count)
      if (x[j] > best) {
        best = x[j];
        at = i + j;
      }
      low = x[j] > -INFINITY ? fminf(low, x[j]) : low;
    }
  }
  uint64_t top = at >= 0 ? rank_of(best, at) : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t t = (uint64_t)__shfl_xor((unsigned long long)top, o, 64);
    top = t > top ? t : top;
    low = fminf(low, __shfl_xor(low, o, 64));
  }
  if ((tid & 63) == 0) {
    sh.tops[tid >> 6] = top;
    sh.lows[tid >> 6] = low;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSampleWaves; ++i) {
      top = sh.tops[i] > top ? sh.tops[i] : top;
      low = fminf(low, sh.lows[i]);
    }
    SampleSeg& out = a.part[(int64_t)r * a.segs + seg];
    out.top = top;
    out.low = low;
    if (seg == 0) a.listed[r] = 0u;
  }
}

// What a row's segments have found, together.
struct SampleWhole {
  uint64_t top, all, before, weight;
  float low;
};
// (every wavefront by itself; all that is asked for is read at once)
template <bool ALL, bool PARTS>
__device__ __forceinline__ SampleWhole over_segments(const SampleArgs& a, int r) {
  SampleWhole v{0, 0, 0, 0, INFINITY};
  for (int s = threadIdx.x & 63; s < a.segs; s += 64) {
    const SampleSeg part = a.part[(int64_t)r * a.segs + s];
    v.top = part.top > v.top ? part.top : v.top;
    v.low = fminf(v.low, part.low);
    if (ALL) v.all += part.all;
    if (PARTS) {
      v.before += part.before;
      v.weight += part.weight;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t t = (uint64_t)__shfl_xor((unsigned long long)v.top, o, 64);
    v.top = t > v.top ? t : v.top;
    v.low = fminf(v.low, __shfl_xor(v.low, o, 64));
    if (ALL) v.all += (uint64_t)__shfl_xor((unsigned long long)v.all, o, 64);
    if (PARTS) {
      v.before += (uint64_t)__shfl_xor((unsigned long long)v.before, o, 64);
      v.weight += (uint64_t)__shfl_xor((unsigned long long)v.weight, o, 64);
    }
  }
  return v;
}

// The row's weights, from its largest and smallest logits and its temperature.  False where there is nothing to sample: `token`
// is then the row's answer.
__device__ __forceinline__ bool row_weights(const SampleWhole& whole, double t, const double* table, SampleWeight& of, int64_t& token) {
  token = whole.top == 0 ? -1 : (int64_t)(kNoIndex - (uint32_t)whole.top);
  if (whole.top == 0 || !(t > 0.0)) return false;
  of.top = (double)float_of((uint32_t)(whole.top >> 32));
  of.infinite = of.top == INFINITY;
  of.c = fmin(1.4426950408889634 / t, 1e300);  // (finite: 0 times it is 0)
  of.table = table;
  const uint64_t most = 44ull << 40, range = of.infinite ? 0u : of.octaves(whole.low);  // (weights below 2^-44 are 0)
  const double scale = (double)(kSampleBins * kSampleInside) * 0x1p32 / (double)((range < most ? range : most) / 16384 + 1);
  of.scale = scale < 4294967295.0 ? (uint32_t)scale : 0xffffffffu;
  return true;
}
__device__ __forceinline__ double row_t(const SampleArgs& a, int r) { return row_value(a.temperature, a.t_s, a.t0, r); }
// A row without borders.
__device__ __forceinline__ SampleRow plain_row(const SampleArgs& a, int r, const SampleWhole& whole) {
  const double given = row_value(a.min_p, a.m_s, a.m0, r), min_p = given >= 1.0 ? 1.0 : given;  // (NaN: no filter)
  SampleRow row{0.0, 0.0, 50ull << 40, -2, 0u, kSampleBins, -1, -1, 0u, 0};
  SampleWeight of;
  int64_t token;
  if (!row_weights(whole, row_t(a, r), nullptr, of, token)) {
    row.token = token;
    return row;
  }
  row.top = of.top;
  row.c = of.c;
  row.scale = of.scale;
  if (min_p > 0x1p-49) row.lightest = (uint64_t)(-log2(min_p) * 0x1p40 + 0.5);
  return row;
}

__device__ __forceinline__ uint64_t part(double p, uint64_t weight) {  // the weight that top-p asks for, at least one unit
  const double x = ceil(p * (double)weight);
  return x >= 1.0 ? (uint64_t)x : 1u;
}
__device__ __forceinline__ int64_t row_k(const SampleArgs& a, int r) {
  const int64_t k = !a.top_k ? a.k0
                    : a.k64  ? reinterpret_cast<const int64_t*>(a.top_k)[r * a.k_s]
                             : (int64_t) reinterpret_cast<const int32_t*>(a.top_k)[r * a.k_s];
  return k > 0 && k < a.vocab ? k : 0;  // 0: all
}
__device__ __forceinline__ double row_p(const SampleArgs& a, int r) {
  const double p = row_value(a.top_p, a.p_s, a.p0, r);
  return p < 1.0 ? p : 1.0;  // 1 (and NaN): all
}

// ------------------------------------------------------------------------------ weights by their size ----
template <typename T>
__device__ __forceinline__ void bins_step(const SampleArgs& a, int seg, int r, double* table, uint64_t* waves, SampleBins& sh) {
  const int tid = threadIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  const int end = (seg + 1) * a.seg < a.vocab ? (seg + 1) * a.seg : a.vocab;
  float next[8];  // (on their way while the row's settings are)
  eight_logits<T>(row, seg * a.seg + 8 * tid, a.vocab, next);
  fill_table(table);
  for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.bins[i] = 0u;
  const int64_t k = row_k(a, r);
  const double p = row_p(a, r);
  SampleWeight of;
  int64_t token;
  if (!row_weights(over_segments<false, false>(a, r), row_t(a, r), table, of, token) || (k == 0 && p == 1.0)) return;
  __syncthreads();
  uint64_t sum = 0;
  for (int i = seg * a.seg + 8 * tid; i < end; i += 8 * kSampleThreads) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = next[j];
    if (i + 8 * kSampleThreads < end) eight_logits<T>(row, i + 8 * kSampleThreads, a.vocab, next);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint64_t y = of.octaves(x[j]), units = of.units(y);
      const uint32_t place = of.place(y);
      sum += units;
      if (units != 0) atomicAdd(&sh.bins[place / kSampleInside], 1u << kSamplePlace | place % kSampleInside);
    }
  }
  sum = block_sum64(sum, waves);
  const int64_t at = (int64_t)r * a.segs + seg;
  if (tid == 0) a.part[at].all = sum;
  static_assert(kSampleBins == 4 * kSampleThreads, "four bins a thread");
  *reinterpret_cast<u32x4_t*>(a.bins + at * kSampleBins + 4 * tid) = *reinterpret_cast<const u32x4_t*>(sh.bins + 4 * tid);
}

__device__ __forceinline__ SampleRow join_step(const SampleArgs& a, int r, SampleJoin& sh) {
  const int tid = threadIdx.x;
  const uint64_t k = (uint64_t)row_k(a, r);
  const double p = row_p(a, r);
  // four bins a thread: their tokens, and bounds of their weights
  uint32_t n[4] = {0u, 0u, 0u, 0u}, places[4] = {0u, 0u, 0u, 0u};
#pragma unroll 8
  for (int g = 0; g < a.segs; ++g) {
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(a.bins + ((int64_t)r * a.segs + g) * kSampleBins + 4 * tid);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      n[i] += v[i] >> kSamplePlace;
      places[i] += v[i] & ((1u << kSamplePlace) - 1u);
    }
  }
  const SampleWhole whole = over_segments<true, false>(a, r);
  SampleRow row = plain_row(a, r, whole);
  if (row.token != -2 || (k == 0 && p == 1.0)) return row;  // (there are no bins)
  // A token of place i has y in [i w, (i + 1) w + 2^-26), w = 2^6 / scale octaves.  2^-y is convex: the sum over tokens whose
  // places have the mean f is at most the chord's from place 0 to the last, and at least their number times the value at f + 1.
  const double width = 64.0 / (double)row.scale;
  uint64_t least[4], most[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double c = (double)n[i], at = (double)((4 * tid + i) * kSampleInside), f = (double)places[i];
    // (32-bit powers of arguments below 64: 2^-24 64 ln 2 of the argument's rounding and 2^-22 of their own, less than 1e-5)
    const double w0 = __builtin_amdgcn_exp2f((float)(43.0 - at * width)), w1 = __builtin_amdgcn_exp2f((float)(43.0 - (at + (kSampleInside - 1)) * width));
    const double high = (c * w0 + (w1 - w0) * f * (1.0 / (kSampleInside - 1))) * 1.00001 + c;  // (and half a unit's rounding each)
    const double mean = f * (double)(1.f / (float)n[i]) * 1.0000003;
    const double low = n[i] ? c * (double)__builtin_amdgcn_exp2f((float)(43.0 - (at + mean + 1.0) * width)) * 0.99999 - c : 0.0;
    least[i] = low > 0.0 ? (uint64_t)low : 0u;
    most[i] = n[i] ? (uint64_t)high + 1u : 0u;
  }
  // the sums of all three in front of this thread, and all tokens
  const uint64_t own[3] = {(uint64_t)n[0] + n[1] + n[2] + n[3], least[0] + least[1] + least[2] + least[3], most[0] + most[1] + most[2] + most[3]};
  uint64_t front[3], total_n = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    front[i] = wave_scan64(own[i]);
    if ((tid & 63) == 63) sh.waves[i][tid >> 6] = front[i];
    front[i] -= own[i];
  }
  if (tid < 3) sh.found[tid] = kSampleBins - 1;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    total_n += sh.waves[0][w];
#pragma unroll
    for (int i = 0; i < 3; ++i) front[i] += w < (tid >> 6) ? sh.waves[i][w] : 0u;
  }
  const uint64_t nb = front[0], lb = front[1], mb = front[2];
  const bool by_k = k > 0 && k < total_n;
  if (by_k) {  // the bin of the k-th token
    uint64_t x = nb, low = lb, high = mb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (x < k && k <= x + n[i]) {
        sh.found[0] = 4 * tid + i;
        sh.bounds[0] = low;
        sh.bounds[1] = high + most[i];
        sh.count = (uint32_t)x;
      }
      x += n[i];
      low += least[i];
      high += most[i];
    }
  }
  __syncthreads();
  const int bk = by_k ? sh.found[0] : -1;
  int plo = by_k ? bk : kSampleBins, phi = by_k ? bk : -1;
  if (p < 1.0) {  // the bins that can have the border
    const uint64_t first = part(p, by_k ? sh.bounds[0] : whole.all), last = part(p, by_k ? sh.bounds[1] : whole.all);
    uint64_t low = lb, high = mb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (high < first && high + most[i] >= first) sh.found[1] = 4 * tid + i;
      if (low < last && low + least[i] >= last) sh.found[2] = 4 * tid + i;
      low += least[i];
      high += most[i];
    }
    __syncthreads();
    plo = sh.found[1] < plo ? sh.found[1] : plo;
    phi = by_k && bk < sh.found[2] ? bk : sh.found[2];
    if (phi < plo) phi = plo;
  }
  row.plo = plo;
  row.phi = phi;
  row.bk = bk;
  row.count = by_k ? sh.count : 0u;
  return row;
}

// ---------------------------------------------------------------------------- the border and the token ----
// A row that all lanes have, in scalar registers.
__device__ __forceinline__ SampleRow alike(const SampleRow& row) {
  constexpr int kWords = sizeof(SampleRow) / 4;
  struct Words {
    uint32_t word[kWords];
  };
  Words words = __builtin_bit_cast(Words, row);
#pragma unroll
  for (int i = 0; i < kWords; ++i) words.word[i] = __builtin_amdgcn_readfirstlane(words.word[i]);
  return __builtin_bit_cast(SampleRow, words);
}
__device__ __forceinline__ bool at_border(const SampleRow& row, int bin) { return (bin >= row.plo && bin <= row.phi) || bin == row.bk; }
__device__ __forceinline__ SampleWeight weights_of(const SampleRow& row, const double* table) {
  return SampleWeight{row.top, row.c, row.top == INFINITY, row.scale, table};
}

// FILTERS: there is a top-k or a top-p.  row_of() gives the row's borders.
template <typename T, bool FILTERS, typename RowOf>
__device__ __forceinline__ void sums_step(const SampleArgs& a, int seg, int r, RowOf row_of, double* table, uint64_t* waves, SampleSums& sh) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  const int end = (seg + 1) * a.seg < a.vocab ? (seg + 1) * a.seg : a.vocab;
  float x[8];  // (on their way while the row's settings are)
  eight_logits<T>(row, seg * a.seg + kSampleSub * w + 8 * lane, a.vocab, x);
  fill_table(table);
  if (tid == 0) sh.met = 0u;
  const SampleRow border = alike(row_of());
  if (border.token != -2) return;
  const SampleWeight of = weights_of(border, table);
  __syncthreads();
  uint64_t before = 0, weight = 0;
  for (int s0 = seg * a.seg + kSampleSub * w; s0 < end; s0 += kSampleWaves * kSampleSub) {
    const int i = s0 + 8 * lane;
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint64_t y = of.octaves(x[j]), units = of.units(y);
      if (!FILTERS) {
        sum += y <= border.lightest ? units : 0u;
        continue;
      }
      const int bin = of.bin(y);
      const uint64_t mine = bin < border.plo ? units : 0u;
      before += mine;
      sum += y <= border.lightest ? mine : 0u;
      if (border.bk >= 0) weight += bin < border.bk ? units : 0u;
      if (at_border(border, bin) && units != 0) {
        const uint32_t at = atomicAdd(&sh.met, 1u);
        if (at < kSampleList) sh.item[at] = rank_of(x[j], i + j);
      }
    }
    sum = wave_sum64(sum);
    if (lane == 0) a.sub[(int64_t)r * a.subs + s0 / kSampleSub] = sum;
    if (s0 + kSampleWaves * kSampleSub < end) eight_logits<T>(row, i + kSampleWaves * kSampleSub, a.vocab, x);
  }
  if (!FILTERS) return;
  __syncthreads();
  uint32_t ready = 0u;  // (the sums go on while it comes)
  if (tid == 0 && sh.met > 0) ready = __hip_atomic_fetch_add(&a.listed[r], sh.met, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  before = block_sum64(before, waves);
  weight = block_sum64(weight, waves);
  SampleSeg& out = a.part[(int64_t)r * a.segs + seg];
  if (tid == 0) {
    out.before = before;
    out.weight = weight;
    sh.ready = ready;
  }
  __syncthreads();
  for (uint32_t i = tid; i < sh.met && i < kSampleList && sh.ready < kSampleList - i; i += kSampleThreads)  // in any order
    a.list[(int64_t)r * kSampleList + sh.ready + i] = sh.item[i];
}

// The list in its order, by buckets of weights (a bucket a thread) and the ranks inside of them: up to 978 tokens, 64 rows of 131072,
// 11.3 us for the whole step, 20.8 where pairs are exchanged.  False, and the list as it was, where a bucket has many tokens.
__device__ __forceinline__ bool sort_by_weight(const SampleArgs& a, int r, uint32_t listed, uint64_t some, const SampleWeight& of,
                                               const SampleRow& border, uint64_t* waves, SampleFinish& sh) {
  constexpr int kPer = kSampleList / kSampleThreads;
  constexpr uint32_t kMany = 64;
  const int tid = threadIdx.x;
  uint32_t* const counts = reinterpret_cast<uint32_t*>(sh.other);
  uint32_t* const starts = counts + kSampleThreads;
  // eighths of places; bins plo to phi have the first buckets, bin bk behind them has one for each of its eighths
  constexpr uint32_t kBin = 8 * kSampleInside;
  const uint32_t first = border.bk > border.phi ? kSampleThreads - kBin : kSampleThreads;
  const uint32_t lo = (uint32_t)border.plo * kBin, range = (uint32_t)(border.phi + 1 - border.plo) * kBin;
  counts[tid] = 0u;
  __syncthreads();
  uint64_t item[kPer];
  uint32_t bucket[kPer], at[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int x = tid + kSampleThreads * i;
    if (x >= (int)listed) break;
    item[i] = i == 0 ? some : a.list[(int64_t)r * kSampleList + x];
    const uint64_t y = of.octaves(float_of((uint32_t)(item[i] >> 32)));
    const uint32_t eighth = (uint32_t)((uint64_t)(uint32_t)(y >> 14) * of.scale >> 29);
    const bool behind = of.bin(y) > border.phi;
    const uint32_t to = behind ? first + eighth - (uint32_t)border.bk * kBin : (eighth - lo) * first / range, end = behind ? kSampleThreads : first;
    bucket[i] = to < end ? to : end - 1;
    at[i] = atomicAdd(&counts[bucket[i]], 1u);
  }
  __syncthreads();
  const uint32_t mine = counts[tid];
  if (__syncthreads_or(mine > kMany)) return false;
  uint64_t all;
  starts[tid] = (uint32_t)block_scan64(mine, waves, all);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (tid + kSampleThreads * i < (int)listed) sh.item[starts[bucket[i]] + at[i]] = item[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (tid + kSampleThreads * i >= (int)listed) break;
    const uint32_t start = starts[bucket[i]], end = start + counts[bucket[i]];
    at[i] = start;
    for (uint32_t x = start; x < end; ++x) at[i] += sh.item[x] > item[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (tid + kSampleThreads * i < (int)listed) sh.item[at[i]] = item[i];
  __syncthreads();
  return true;
}

template <typename T>
__device__ __forceinline__ void finish_step(const SampleArgs& a, int r, double* table, uint64_t* waves, SampleFinish& sh) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  // what is read from memory goes out together: a wait for one after another is most of a small row's time
  const uint32_t listed = a.listed[r];
  const uint64_t some = a.list[(int64_t)r * kSampleList + tid];  // (its place exists; looked at up to `listed`)
  const double u = (double)a.u[r * a.u_s];
  fill_table(table);
  for (int i = tid; i < a.subs; i += kSampleThreads) sh.sub[i] = a.sub[(int64_t)r * a.subs + i];
  const double p = row_p(a, r);
  const uint64_t k = (uint64_t)row_k(a, r);
  const SampleWhole whole = over_segments<true, true>(a, r);  // (before and weight are there where there are filters)
  const SampleRow border = a.filters ? a.row[r] : plain_row(a, r, whole);
  if (border.token != -2) {  // nothing to choose from, or nothing to choose
    if (tid == 0) a.out[r] = border.token;
    return;
  }
  const SampleWeight of = weights_of(border, table);
  const bool fits = listed <= kSampleList;
  __syncthreads();
  uint64_t least = 0;  // the rank of the last token that stays
  if (listed > 0) {
    const int bk = border.bk, phi = border.phi;
    const uint64_t want_k = bk >= 0 ? k - border.count : 0;  // tokens of bin bk that stay
    const uint64_t in_front_of_plo = whole.before;
    uint64_t total = bk >= 0 ? whole.weight : whole.all;
    if (fits) {
      // the list from the largest rank down
      if (listed > kSampleCounted && sort_by_weight(a, r, listed, some, of, border, waves, sh)) {
      } else if (listed <= kSampleThreads) {  // a token a thread, to the place behind all larger ones
        sh.other[tid] = tid < (int)listed ? some : 0u;
        __syncthreads();
        int at = 0;
        for (int i = 0; i < (int)listed; i += 4)  // (zeros behind the list)
#pragma unroll
          for (int j = 0; j < 4; ++j) at += sh.other[i + j] > some;
        if (tid < (int)listed) sh.item[at] = some;
        __syncthreads();
      } else {  // in pairs, and zeros behind it
        int n = 2 * kSampleThreads;
        while (n < (int)listed) n *= 2;
        for (int i = tid; i < n; i += kSampleThreads)
          sh.item[i] = i >= (int)listed ? 0u : (i == tid ? some : a.list[(int64_t)r * kSampleList + i]);
        __syncthreads();
        for (int size = 2; size <= n; size *= 2)
          for (int step = size / 2; step > 0; step /= 2) {
            for (int i = tid; i < n / 2; i += kSampleThreads) {
              const int x = 2 * i - (i & (step - 1)), z = x + step;
              const uint64_t p0 = sh.item[x], p1 = sh.item[z];
              if ((p0 < p1) == ((x & size) == 0)) {
                sh.item[x] = p1;
                sh.item[z] = p0;
              }
            }
            // up to steps of 64 a wavefront stays within 128 tokens of its own
            if (step > 64 || (step == 1 && size >= 128)) {
              __syncthreads();
            } else {
              __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
              __builtin_amdgcn_wave_barrier();
            }
          }
        __syncthreads();
      }
      // running sums: of four tokens a thread
      constexpr int kPer = kSampleList / kSampleThreads;
      uint64_t units[kPer], upto[kPer], y[kPer], all;
      int in_front = 0, in_range = 0;  // tokens in bins in front of bk; in bins up to phi
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = kPer * tid + i;
        const bool there = at < (int)listed;
        y[i] = there ? of.octaves(float_of((uint32_t)(sh.item[at] >> 32))) : 0u;
        units[i] = there ? of.units(y[i]) : 0u;
        const int bin = of.bin(y[i]);
        in_front += there && bin < bk;
        in_range += there && bin <= phi;
      }
      uint64_t sum = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum += units[i];
      uint64_t before = block_scan64(sum, waves, all);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        upto[i] = before;
        before += units[i];
      }
      const uint64_t counts = block_sum64((uint64_t)in_front << 32 | (uint32_t)in_range, waves);
      const int front = (int)(counts >> 32), range = (int)(uint32_t)counts;
      int cut = (int)listed;  // tokens of the list that stay
      if (bk >= 0) {
        cut = front + (int)want_k;
        uint64_t s = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) s += kPer * tid + i >= front && kPer * tid + i < cut ? units[i] : 0u;
        total += block_sum64(s, waves);
      }
      if (p < 1.0) {
        const uint64_t want = part(p, total);
        const int most = range < cut ? range : cut;
        uint64_t s = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) s += kPer * tid + i < most && in_front_of_plo + upto[i] < want;
        cut = (int)block_sum64(s, waves);  // (the border may be the end of bin phi: what is behind it goes)
      }
      least = sh.item[cut > 0 ? cut - 1 : 0];  // (at least one: less weight than asked for is in front of bin plo)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = kPer * tid + i;
        if (at < cut && y[i] <= border.lightest)
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.sub[(kNoIndex - (uint32_t)sh.item[at]) / kSampleSub]), (unsigned long long)units[i]);
      }
    } else {
      // f(rank, y, bin) of this thread's share of the border's tokens, and its sum over all of them
      auto each = [&](auto f) {
        for (int i = 8 * tid; i < a.vocab; i += 8 * kSampleThreads) {
          float x[8];
          eight_logits<T>(row, i, a.vocab, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint64_t y = of.octaves(x[j]);
            const int bin = of.bin(y);
            if (at_border(border, bin) && of.units(y) != 0) f(rank_of(x[j], i + j), y, bin);
          }
        }
      };
      auto sum_of = [&](auto f) {
        uint64_t s = 0;
        each([&](uint64_t rank, uint64_t y, int bin) { s += f(rank, y, bin); });
        return block_sum64(s, waves);
      };
      unsigned long long* const ends = reinterpret_cast<unsigned long long*>(sh.item);  // the smallest and the largest rank
      if (tid == 0) {
        ends[0] = ~0ull;
        ends[1] = 0;
      }
      __syncthreads();
      uint64_t smallest = ~0ull, most = 0;
      each([&](uint64_t rank, uint64_t, int) {
        smallest = rank < smallest ? rank : smallest;
        most = rank > most ? rank : most;
      });
      if (most > 0) {
        atomicMin(&ends[0], (unsigned long long)smallest);
        atomicMax(&ends[1], (unsigned long long)most);
      }
      __syncthreads();
      // the largest rank x with f(x), which holds at the smallest and, where it holds, for everything smaller
      auto largest = [&](auto f) {
        uint64_t lo = ends[0], hi = ends[1];
        while (lo < hi) {
          const uint64_t mid = lo + (hi - lo) / 2 + 1;
          if (f(mid)) lo = mid;
          else hi = mid - 1;
        }
        return lo;
      };
      if (bk >= 0) {
        least = largest([&](uint64_t x) {
          return sum_of([&](uint64_t rank, uint64_t, int bin) { return (uint64_t)(bin == bk && rank >= x); }) >= want_k;
        });
        total += sum_of([&](uint64_t rank, uint64_t y, int bin) { return bin == bk && rank >= least ? of.units(y) : 0ull; });
      }
      if (p < 1.0) {
        const uint64_t want = part(p, total), stays = least;
        const auto upto = [&](uint64_t x) {  // weight of the tokens with ranks of at least x
          return in_front_of_plo + sum_of([&](uint64_t rank, uint64_t y, int bin) { return bin <= phi && rank >= x && rank >= stays ? of.units(y) : 0ull; });
        };
        if (upto(0) >= want) least = largest([&](uint64_t x) { return upto(x) >= want; });
      }
      for (int s0 = kSampleSub * w; s0 < a.vocab; s0 += kSampleWaves * kSampleSub) {
        float x[8];
        const int i = s0 + 8 * lane;
        eight_logits<T>(row, i, a.vocab, x);
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint64_t y = of.octaves(x[j]);
          if (y <= border.lightest && rank_of(x[j], i + j) >= least) sum += of.units(y);
        }
        sum = wave_sum64(sum);
        if (lane == 0) sh.sub[s0 / kSampleSub] = sum;
      }
    }
  }
  __syncthreads();
  // which of them the random number falls into
  constexpr int kPer = kSampleSubs / kSampleThreads;
  uint64_t mine[kPer], sum = 0, all;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mine[i] = kPer * tid + i < a.subs ? sh.sub[kPer * tid + i] : 0u;
    sum += mine[i];
  }
  uint64_t before = block_scan64(sum, waves, all);
  const double aim = u > 0.0 ? floor(u * (double)all) : 0.0;  // (a NaN: 0)
  uint64_t target = aim < (double)all ? (uint64_t)aim : all - 1;
  if (target >= all) target = all - 1;  // (a sum that its double is larger than)
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (before <= target && target < before + mine[i]) {
      sh.chosen = kPer * tid + i;
      sh.left = target - before;
    }
    before += mine[i];
  }
  __syncthreads();
  if (w != 0) return;
  const int i0 = kSampleSub * sh.chosen + 8 * lane;
  const uint64_t left = sh.left;
  float x[8];
  eight_logits<T>(row, i0, a.vocab, x);
  uint64_t units[8];
  sum = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint64_t y = of.octaves(x[j]);
    units[j] = y <= border.lightest && rank_of(x[j], i0 + j) >= least ? of.units(y) : 0u;
    sum += units[j];
  }
  uint64_t upto = wave_scan64(sum) - sum;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (upto <= left && left < upto + units[j]) a.out[r] = i0 + j;
    upto += units[j];
  }
}

// --------------------------------------------------------------------------------------- launches ----
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_top(SampleArgs a) {
  __shared__ SampleTop sh;
  top_step<T>(a, blockIdx.x % a.segs, blockIdx.x / a.segs, sh);
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_bins(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) double table[kSampleTable];
  __shared__ uint64_t waves[kSampleWaves];
  __shared__ __attribute__((aligned(16))) SampleBins sh;
  bins_step<T>(a, blockIdx.x % a.segs, blockIdx.x / a.segs, table, waves, sh);
}
__global__ __launch_bounds__(kSampleThreads) void sample_join(SampleArgs a) {
  __shared__ SampleJoin sh;
  const SampleRow row = join_step(a, blockIdx.x, sh);
  if (threadIdx.x == 0) a.row[blockIdx.x] = row;
}
// (registers for four workgroups a compute unit: with the next tokens' loads ahead of time they allow two, 64 x 131072 in 23.4 us
// instead of 19.5)
template <typename T, bool FILTERS>
__global__ __launch_bounds__(kSampleThreads, 8) void sample_sums(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) double table[kSampleTable];
  __shared__ uint64_t waves[kSampleWaves];
  __shared__ SampleSums sh;
  const int r = blockIdx.x / a.segs;
  auto row_of = [&] { return FILTERS ? a.row[r] : plain_row(a, r, over_segments<false, false>(a, r)); };
  sums_step<T, FILTERS>(a, blockIdx.x % a.segs, r, row_of, table, waves, sh);
}
// join and sums in one launch: every workgroup joins its row's bins.
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_join_sums(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) double table[kSampleTable];
  __shared__ uint64_t waves[kSampleWaves];
  __shared__ SampleJoin join;
  __shared__ SampleSums sh;
  const int r = blockIdx.x / a.segs, seg = blockIdx.x % a.segs;
  auto row_of = [&] {
    const SampleRow row = join_step(a, r, join);
    if (seg == 0 && threadIdx.x == 0) a.row[r] = row;
    return row;
  };
  sums_step<T, true>(a, seg, r, row_of, table, waves, sh);
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_finish(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) double table[kSampleTable];
  __shared__ uint64_t waves[kSampleWaves];
  __shared__ SampleFinish sh;
  finish_step<T>(a, blockIdx.x, table, waves, sh);
}
// All steps of a row that is one segment, by one workgroup, which sees its own writes behind a barrier.
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_whole(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) SampleShared sh;
  const int r = blockIdx.x;
  top_step<T>(a, 0, r, sh.top);
  __syncthreads();
  if (a.filters) {
    bins_step<T>(a, 0, r, sh.table, sh.waves, sh.bins);
    __syncthreads();
    const SampleRow row = join_step(a, r, sh.join);
    if (threadIdx.x == 0) a.row[r] = row;
    __syncthreads();
    sums_step<T, true>(a, 0, r, [&] { return a.row[r]; }, sh.table, sh.waves, sh.sums);
  } else {
    sums_step<T, false>(a, 0, r, [&] { return plain_row(a, r, over_segments<false, false>(a, r)); }, sh.table, sh.waves, sh.sums);
  }
  __syncthreads();
  finish_step<T>(a, r, sh.table, sh.waves, sh.finish);
}

// Tokens of a workgroup: enough workgroups for the card where there are that many tokens, at most kSampleSeg.
static int sample_seg(int64_t rows, int64_t vocab) {
  constexpr int64_t step = kSampleWaves * kSampleSub;
  return vocab > step && rows * vocab > 512 * step ? kSampleSeg : (int)step;
}

struct SampleSpace {
  int64_t row, part, sub, list, bins, listed, bytes;
};
static SampleSpace sample_space(int64_t rows, int64_t vocab, int64_t seg) {
  const int64_t segs = cdiv(vocab, seg), subs = cdiv(vocab, kSampleSub);
  SampleSpace s;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t x = at;
    at += (bytes + 15) & ~INT64_C(15);  // (16-byte loads)
    return x;
  };
  s.row = take(rows * sizeof(SampleRow));
  s.part = take(rows * segs * sizeof(SampleSeg));
  s.sub = take(rows * subs * 8);
  s.list = take(rows * kSampleList * 8);
  s.bins = take(rows * segs * kSampleBins * 4);
  s.listed = take(rows * 4);
  s.bytes = at;
  return s;
}
// Rows that go through the launches together: a row has 16 KB of list and 8 KB of bins for each segment, which would be gigabytes for
// many rows.  Half a gigabyte is 3600 rows of 131072 tokens or 21800 short ones: many rounds of workgroups in every launch.
constexpr int64_t kSampleSpace = INT64_C(1) << 29;
static int64_t sample_rows(int64_t rows, int64_t vocab) {
  const int64_t most = kSampleSpace / sample_space(1, vocab, sample_seg(rows, vocab)).bytes;
  return cdiv(rows, cdiv(rows, most));
}

// Workgroups up to which each joins its row's bins itself: one launch less for bins that each of them reads.  us (joined /
// apart): one row of 32000 10.5 / 6.2 + 5.6, 8 of 131072 (256 workgroups) 15.2 / 9.5 + 7.3, 16 21.0 / 9.4 + 10.6, 64 38.8 / 7.6 + 18.7.
constexpr int kSampleJoined = 256;

template <typename T>
static int sample_launch(const SampleArgs& a, hipStream_t s) {
  const dim3 rows((unsigned)a.rows), all((unsigned)(a.rows * a.segs)), threads(kSampleThreads);
  if (a.segs == 1) {
    hipLaunchKernelGGL((sample_whole<T>), rows, threads, 0, s, a);
    return check_launch("sample_whole");
  }
  hipLaunchKernelGGL((sample_top<T>), all, threads, 0, s, a);
  if (const int rc = check_launch("sample_top")) return rc;
  if (a.filters) {
    hipLaunchKernelGGL((sample_bins<T>), all, threads, 0, s, a);
    if (const int rc = check_launch("sample_bins")) return rc;
    if (a.rows * a.segs <= kSampleJoined) {
      hipLaunchKernelGGL((sample_join_sums<T>), all, threads, 0, s, a);
      if (const int rc = check_launch("sample_join_sums")) return rc;
    } else {
      hipLaunchKernelGGL(sample_join, rows, threads, 0, s, a);
      if (const int rc = check_launch("sample_join")) return rc;
      hipLaunchKernelGGL((sample_sums<T, true>), all, threads, 0, s, a);
      if (const int rc = check_launch("sample_sums")) return rc;
    }
  } else {
    hipLaunchKernelGGL((sample_sums<T, false>), all, threads, 0, s, a);
    if (const int rc = check_launch("sample_sums")) return rc;
  }
  hipLaunchKernelGGL((sample_finish<T>), rows, threads, 0, s, a);
  return check_launch("sample_finish");
}

}  // namespace biops

using namespace biops;

extern "C" int64_t biops_sample_workspace_size(int64_t rows, int64_t vocab) {
  if (rows < 0 || vocab < 1 || vocab > kSampleMost || rows > 65536 || rows * vocab > kSampleAll) return -1;
  return rows == 0 ? 0 : sample_space(sample_rows(rows, vocab), vocab, sample_seg(rows, vocab)).bytes;
}

extern "C" int biops_sample(int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const float* u, int64_t u_s,
                            const float* temperature, int64_t t_s, double t0, const void* top_k, int k64, int64_t k_s, int64_t k0,
                            const float* top_p, int64_t p_s, double p0, const float* min_p, int64_t m_s, double m0, int64_t* out,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  if (!is_float_dtype(dtype)) return fail(BIOPS_ERR_DTYPE, "biops_sample: unsupported dtype %d", dtype);
  if (rows < 0 || rows > 65536 || vocab < 1 || vocab > kSampleMost || rows * vocab > kSampleAll)
    return fail(BIOPS_ERR_ARG, "biops_sample: rows of 1 to %d tokens, at most 65536 rows and 2^35 tokens in all", kSampleMost);
  if (rows == 0) return BIOPS_OK;
  if (!logits || !u || !out) return fail(BIOPS_ERR_ARG, "biops_sample: null pointer");
  const int64_t some = sample_rows(rows, vocab);
  const SampleSpace x = sample_space(some, vocab, sample_seg(rows, vocab));
  if (!workspace || workspace_bytes < x.bytes)
    return fail(BIOPS_ERR_SIZE, "biops_sample: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)x.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BIOPS_ERR_LAYOUT, "biops_sample: workspace not 16-byte aligned");
  SampleArgs a;
  a.logits = static_cast<const char*>(logits), a.ld = dtype_bytes(dtype) * ld;
  a.u = u, a.temperature = temperature, a.top_p = top_p, a.min_p = min_p, a.top_k = top_k;
  a.u_s = u_s, a.t_s = t_s, a.k_s = k_s, a.p_s = p_s, a.m_s = m_s;
  a.t0 = t0, a.p0 = p0, a.m0 = m0, a.k0 = k0, a.k64 = k64 != 0;
  a.filters = top_k || top_p || (k0 > 0 && k0 < vocab) || p0 < 1.0;
  a.vocab = (int)vocab;
  a.seg = sample_seg(rows, vocab), a.segs = (int)cdiv(vocab, a.seg), a.subs = (int)cdiv(vocab, kSampleSub);
  char* const base = static_cast<char*>(workspace);
  a.row = reinterpret_cast<SampleRow*>(base + x.row), a.part = reinterpret_cast<SampleSeg*>(base + x.part);
  a.sub = reinterpret_cast<uint64_t*>(base + x.sub), a.list = reinterpret_cast<uint64_t*>(base + x.list);
  a.bins = reinterpret_cast<uint32_t*>(base + x.bins), a.listed = reinterpret_cast<uint32_t*>(base + x.listed);
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t r = 0; r < rows; r += some) {  // one after another in the same workspace
    a.rows = (int)(rows - r < some ? rows - r : some);
    a.logits = static_cast<const char*>(logits) + r * a.ld, a.out = out + r;
    a.u = u + r * u_s;
    if (temperature) a.temperature = temperature + r * t_s;
    if (top_p) a.top_p = top_p + r * p_s;
    if (min_p) a.min_p = min_p + r * m_s;
    if (top_k) a.top_k = static_cast<const char*>(top_k) + r * k_s * (k64 ? 8 : 4);
    int rc = BIOPS_OK;
    BIOPS_DISPATCH_FLOAT(dtype, rc = sample_launch<T>(a, s));
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}

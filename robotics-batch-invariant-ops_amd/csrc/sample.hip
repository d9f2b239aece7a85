// The next token of each row of logits, from one uniform random number a row.
//
// With T the temperature, M the row's largest logit and w_i = exp((l_i - M) / T), tokens are ranked by their logits, equal
// ones by their index.  Of this order stays the beginning that every filter allows: the first k (top-k), those before which
// less than p of the weight of the first k has gone (top-p), those with w_i >= min-p.  The token is the first index whose
// running sum of the weights that stay is past u times all of them.
//
// Sums decide between neighbours, so they are exact: a weight is a 64-bit exponential rounded once to a multiple of 2^-43,
// and sums of those are integers, the same in any order.  A row's token depends on its own row only.
//
// Three launches share a row's tokens among `segs` workgroups.  sample_top finds a segment's largest and smallest logit.
// sample_bins counts tokens and weights in 1024 bins of log2 of the weight; the last workgroup of a row to end adds them up
// and finds the bins that a border can lie in.  sample_pick sums the weights in front of those bins for every 512 tokens and lists
// the tokens inside of them; the last workgroup of a row finds the border in the list (by bisection, first of the logit,
// then of the index among equal ones), completes the sums, and finds the token.  Where the list is too long (thousands of
// tokens in a bin: equal logits) that workgroup reads the row instead, at each step.
//
// What bounds it: the first launch reads the row from memory; then 16 operations in 64 bits a token, twice, and three
// launches with two joins, which is all there is for few rows.
#include "biops_common.h"

namespace biops {

constexpr int kSampleBins = 1024, kSampleList = 2048, kSampleSub = 512;
constexpr int kSampleMost = 1 << 20;           // tokens of a row: sums of that many weights fit 64 bits
constexpr int kSampleSubs = kSampleMost / kSampleSub;
constexpr double kSampleOctaves = 32.0;        // what the bins cover at most, as powers of two of the weight
constexpr uint32_t kNoIndex = 0xffffffffu;

struct SampleRow {
  double c, bins, min_p, p;         // log2 e / T; bins per octave; p >= 1: all
  uint64_t k, weight, before, all;  // k 0: all; weight in front of bin bk, and of plo; of all tokens
  float top;
  int state;                        // 0: to be sampled; 1: done
  int plo, phi, bk;                 // bins of the border of top-p (or of top-k alone), of top-k
  uint32_t count;                   // tokens in front of bin bk
  uint32_t listed;                  // tokens of those bins
  int unused;
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
  int rows, vocab, segs, seg, subs, k64;        // seg: tokens of a workgroup, a multiple of kSampleSub
  // workspace
  SampleRow* row;
  uint64_t *tops, *weights, *sub, *list;        // [rows][segs], [rows][segs][bins], [rows][subs], [rows][kSampleList]
  uint32_t *counts, *ends;                      // [rows][segs][bins]; [rows][3]: workgroups that ended, entries of the list
  float* lows;                                  // [rows][segs]
};

// Larger logits have larger keys; equal ones equal keys.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ bool counts_at_all(float x) { return x > -INFINITY; }  // not -inf, not NaN

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

// The weight 2^-y of a logit in units of 2^-43, with 2^(-i / 64) from a table and the rest by its series: relative error
// below 2^-47.
struct SampleWeight {
  double top, c, bins;
  const double* table;
  __device__ __forceinline__ double octaves(float x) const {
    const double d = top - (double)x;
    return d > 0.0 ? fmin(d * c, 1000.0) : 0.0;  // (0 * inf and inf - inf are 0)
  }
  __device__ __forceinline__ int bin(double y) const {
    const double b = y * bins;
    return b < (double)kSampleBins ? (int)b : kSampleBins - 1;
  }
  __device__ __forceinline__ double weight(double y) const {
    const double z = y * 64.0, whole = floor(z), r = z - whole;
    const int n = (int)whole;
    constexpr double a = 0.010830424696249145;  // ln 2 / 64
    double e = -a * a * a * a * a / 120.0;
    e = fma(e, r, a * a * a * a / 24.0);
    e = fma(e, r, -a * a * a / 6.0);
    e = fma(e, r, a * a / 2.0);
    e = fma(e, r, -a);
    e = fma(e, r, 1.0);
    return ldexp(e * table[n & 63], -(n >> 6));
  }
  __device__ static __forceinline__ uint64_t units(double w) {
    return (uint64_t)__double_as_longlong(w * 0x1p43 + 0x1p52) & 0xfffffffffffffull;  // to the nearest
  }
};
// (a block of at least 64 threads; __syncthreads before use)
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(-(double)threadIdx.x / 64.0);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int from) { return (uint64_t)__shfl((unsigned long long)v, from, 64); }
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, o, 64);
  return v;
}
// Inclusive sums over the wavefront's lanes.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t x = (uint64_t)__shfl_up((unsigned long long)v, o, 64);
    if (lane >= o) v += x;
  }
  return v;
}
// Sum over the 256 threads, to all of them.
__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* four) {
  v = wave_sum64(v);
  __syncthreads();  // (the last sum has been read)
  if ((threadIdx.x & 63) == 0) four[threadIdx.x >> 6] = v;
  __syncthreads();
  return four[0] + four[1] + four[2] + four[3];
}

// Whether this workgroup is the last of `n` that end here: what the others wrote before is then visible to it.
__device__ __forceinline__ bool last_to_end(uint32_t* count, int n, uint32_t* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    *flag = __hip_atomic_fetch_add(count, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(n - 1);
  }
  __syncthreads();
  if (*flag == 0) return false;
  __threadfence();
  return true;
}

__device__ __forceinline__ double row_value(const float* p, int64_t s, double all, int r) { return p ? (double)p[r * s] : all; }

// --------------------------------------------------------------------------------- largest logits ----
template <typename T>
__global__ __launch_bounds__(256) void sample_top(SampleArgs a) {
  __shared__ uint64_t tops[4];
  __shared__ float lows[4];
  const int seg = blockIdx.x % a.segs, r = blockIdx.x / a.segs, tid = threadIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  const int end = (seg + 1) * a.seg < a.vocab ? (seg + 1) * a.seg : a.vocab;
  uint64_t top = 0;  // (key, ~index): 0 where nothing counts
  float best = -INFINITY, low = INFINITY;
  int at = -1;
  for (int i = seg * a.seg + 8 * tid; i < end; i += 2048) {
    float x[8];
    eight_logits<T>(row, i, a.vocab, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!counts_at_all(x[j])) continue;
      if (x[j] > best) {
        best = x[j];
        at = i + j;
      }
      low = fminf(low, x[j]);
    }
  }
  if (at >= 0) top = (uint64_t)key_of(best) << 32 | (kNoIndex - (uint32_t)at);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t t = (uint64_t)__shfl_xor((unsigned long long)top, o, 64);
    top = t > top ? t : top;
    low = fminf(low, __shfl_xor(low, o, 64));
  }
  if ((tid & 63) == 0) {
    tops[tid >> 6] = top;
    lows[tid >> 6] = low;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 4; ++i) {
      top = tops[i] > top ? tops[i] : top;
      low = fminf(low, lows[i]);
    }
    a.tops[(int64_t)r * a.segs + seg] = top;
    a.lows[(int64_t)r * a.segs + seg] = low;
    if (seg == 0)
      for (int i = 0; i < 3; ++i) a.ends[3 * r + i] = 0u;
  }
}

// ------------------------------------------------------------------------------ weights by their size ----
// The row's largest logit and its first index, its smallest, and its settings, from the segments (all threads alike).
__device__ __forceinline__ uint64_t row_top(const SampleArgs& a, int r, float& low) {
  uint64_t top = 0;
  low = INFINITY;
  for (int s = 0; s < a.segs; ++s) {
    const uint64_t t = a.tops[(int64_t)r * a.segs + s];
    top = t > top ? t : top;
    low = fminf(low, a.lows[(int64_t)r * a.segs + s]);
  }
  return top;
}
__device__ __forceinline__ float float_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

__device__ __forceinline__ uint64_t part(double p, uint64_t weight) {  // the weight that top-p asks for, at least one unit
  const double x = ceil(p * (double)weight);
  return x >= 1.0 ? (uint64_t)x : 1u;
}

template <typename T>
__global__ __launch_bounds__(256) void sample_bins(SampleArgs a) {
  __shared__ double table[64];
  __shared__ uint32_t count[kSampleBins];
  __shared__ uint64_t weight[kSampleBins];
  __shared__ uint64_t sums[2][4];
  __shared__ uint32_t last;
  __shared__ int found[3];
  __shared__ uint64_t at_found[2];
  __shared__ uint32_t count_found[2];
  const int seg = blockIdx.x % a.segs, r = blockIdx.x / a.segs, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  float low;
  const uint64_t top = row_top(a, r, low);
  const double t = row_value(a.temperature, a.t_s, a.t0, r);
  const bool greedy = !(t > 0.0);
  if (top == 0 || greedy) {  // nothing to choose from, or nothing to choose
    if (seg == 0 && tid == 0) {
      a.row[r].state = 1;
      a.out[r] = top == 0 ? -1 : (int64_t)(kNoIndex - (uint32_t)top);
    }
    return;
  }
  SampleWeight of;
  of.top = (double)float_of((uint32_t)(top >> 32));
  of.c = 1.4426950408889634 / t;
  of.table = table;
  const bool infinite = of.top == INFINITY;  // only those with the same logit count
  const double range = infinite ? 0.0 : fmin(of.octaves(low), kSampleOctaves);
  of.bins = range > 0.0 ? kSampleBins / range : 0.0;
  fill_table(table);
  for (int i = tid; i < kSampleBins; i += 256) {
    count[i] = 0u;
    weight[i] = 0u;
  }
  __syncthreads();
  const int end = (seg + 1) * a.seg < a.vocab ? (seg + 1) * a.seg : a.vocab;
  for (int i = seg * a.seg + 8 * tid; i < end; i += 2048) {
    float x[8];
    eight_logits<T>(row, i, a.vocab, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!counts_at_all(x[j]) || (infinite && x[j] != INFINITY)) continue;
      const double y = of.octaves(x[j]);
      const uint64_t units = SampleWeight::units(of.weight(y));
      if (units == 0) continue;
      const int b = of.bin(y);
      atomicAdd(&count[b], 1u);
      atomicAdd(reinterpret_cast<unsigned long long*>(&weight[b]), (unsigned long long)units);
    }
  }
  __syncthreads();
  const int64_t mine = ((int64_t)r * a.segs + seg) * kSampleBins;
  for (int i = tid; i < kSampleBins; i += 256) {
    a.counts[mine + i] = count[i];
    a.weights[mine + i] = weight[i];
  }
  if (!last_to_end(&a.ends[3 * r], a.segs, &last)) return;

  // four bins a thread, over all segments
  uint32_t n[4] = {0u, 0u, 0u, 0u};
  uint64_t s[4] = {0u, 0u, 0u, 0u};
  for (int g = 0; g < a.segs; ++g) {
    const int64_t at = ((int64_t)r * a.segs + g) * kSampleBins + 4 * tid;
    const u32x4_t c = *reinterpret_cast<const u32x4_t*>(a.counts + at);
    const u32x4_t w0 = *reinterpret_cast<const u32x4_t*>(a.weights + at), w1 = *reinterpret_cast<const u32x4_t*>(a.weights + at + 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] += c[i];
    s[0] += (uint64_t)w0[1] << 32 | w0[0];
    s[1] += (uint64_t)w0[3] << 32 | w0[2];
    s[2] += (uint64_t)w1[1] << 32 | w1[0];
    s[3] += (uint64_t)w1[3] << 32 | w1[2];
  }
  const uint64_t n4 = n[0] + n[1] + n[2] + n[3], s4 = s[0] + s[1] + s[2] + s[3];
  const uint64_t nscan = wave_scan64(n4), sscan = wave_scan64(s4);
  if (lane == 63) {
    sums[0][w] = nscan;
    sums[1][w] = sscan;
  }
  if (tid < 3) found[tid] = kSampleBins;
  __syncthreads();
  uint64_t nb = nscan - n4, sb = sscan - s4, total_n = 0, total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) {
      nb += sums[0][i];
      sb += sums[1][i];
    }
    total_n += sums[0][i];
    total += sums[1][i];
  }
  int64_t k = a.k0;
  if (a.top_k) k = a.k64 ? reinterpret_cast<const int64_t*>(a.top_k)[r * a.k_s] : (int64_t) reinterpret_cast<const int32_t*>(a.top_k)[r * a.k_s];
  const bool by_k = k > 0 && (uint64_t)k < total_n;
  const double p = row_value(a.top_p, a.p_s, a.p0, r);
  const bool by_p = p < 1.0;  // (a NaN: all)
  if (by_k) {  // the bin of the k-th token
    uint64_t x = nb, y = sb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (x < (uint64_t)k && (uint64_t)k <= x + n[i]) {
        found[0] = 4 * tid + i;
        at_found[0] = y;
        at_found[1] = s[i];
        count_found[0] = (uint32_t)x;
      }
      x += n[i];
      y += s[i];
    }
  }
  __syncthreads();
  const int bk = by_k ? found[0] : -1;
  int plo = by_k ? bk : kSampleBins, phi = by_k ? bk : -1;
  if (by_p) {  // the bins that have the border, whatever part of bin bk counts
    const uint64_t least = part(p, by_k ? at_found[0] : total), most = part(p, by_k ? at_found[0] + at_found[1] : total);
    uint64_t y = sb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t z = y + s[i];
      if (y < least && z >= least) found[1] = 4 * tid + i;
      if (y < most && z >= most) found[2] = 4 * tid + i;
      y = z;
    }
    __syncthreads();
    plo = found[1] < plo ? found[1] : plo;
    phi = by_k ? (found[2] < bk ? found[2] : bk) : found[2];
    if (phi < plo) phi = plo;
  }
  // what is in front of bin plo, and how many tokens the border's bins have
  uint64_t listed = 0;
  {
    uint64_t y = sb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = 4 * tid + i;
      if (b == plo) a.row[r].before = y;
      if ((b >= plo && b <= phi) || b == bk) listed += n[i];
      y += s[i];
    }
  }
  listed = block_sum64(listed, sums[0]);
  if (tid == 0) {
    SampleRow& out = a.row[r];
    out.c = of.c;
    out.bins = of.bins;
    out.min_p = fmin(row_value(a.min_p, a.m_s, a.m0, r), 1.0);
    out.p = by_p ? p : 1.0;
    out.k = by_k ? (uint64_t)k : 0u;
    out.weight = by_k ? at_found[0] : 0u;
    out.all = total;
    out.top = (float)of.top;
    out.state = 0;
    out.plo = plo;
    out.phi = phi;
    out.bk = bk;
    out.count = by_k ? count_found[0] : 0u;
    out.listed = (uint32_t)listed;
  }
}

// ---------------------------------------------------------------------------- the border and the token ----
// A token of the border's bins.
struct SampleItem {
  uint32_t key, index;
  uint64_t units;
  int bin;
  bool heavy;  // enough for min-p
};

template <typename T>
__global__ __launch_bounds__(256) void sample_pick(SampleArgs a) {
  __shared__ double table[64];
  __shared__ uint64_t four[4];
  __shared__ uint32_t last, ready, met;
  __shared__ uint64_t sub[kSampleSubs];
  __shared__ uint32_t item_key[kSampleList], item_index[kSampleList];
  __shared__ uint64_t item_units[kSampleList];
  __shared__ uint16_t item_bin[kSampleList];
  __shared__ int chosen;
  __shared__ uint64_t left;
  const int seg = blockIdx.x % a.segs, r = blockIdx.x / a.segs, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* row = reinterpret_cast<const T*>(a.logits + r * a.ld);
  const SampleRow& in = a.row[r];
  if (in.state != 0) return;
  SampleWeight of;
  of.top = (double)in.top;
  of.c = in.c;
  of.bins = in.bins;
  of.table = table;
  const bool infinite = of.top == INFINITY;
  const int plo = in.plo, phi = in.phi, bk = in.bk;
  const double min_p = in.min_p;
  const bool fits = in.listed <= kSampleList;
  fill_table(table);
  if (tid == 0) met = 0u;
  __syncthreads();
  // (octaves, bin, weight) of a logit; false where it does not count
  auto item_of = [&](float x, uint32_t index, SampleItem& t) {
    if (!counts_at_all(x) || (infinite && x != INFINITY)) return false;
    const double y = of.octaves(x), weight = of.weight(y);
    t.key = key_of(x);
    t.index = index;
    t.units = SampleWeight::units(weight);
    t.bin = of.bin(y);
    t.heavy = !(weight < min_p);
    return t.units != 0;
  };
  auto at_border = [&](int bin) { return (bin >= plo && bin <= phi) || bin == bk; };

  const int end = (seg + 1) * a.seg < a.vocab ? (seg + 1) * a.seg : a.vocab;
  if (fits)
    for (int s0 = seg * a.seg + kSampleSub * w; s0 < end; s0 += 4 * kSampleSub) {
      float x[8];
      const int i = s0 + 8 * lane;
      eight_logits<T>(row, i, a.vocab, x);
      uint64_t sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        SampleItem t;
        if (!item_of(x[j], i + j, t)) continue;
        if (t.bin < plo) {
          if (t.heavy) sum += t.units;
        } else if (at_border(t.bin)) {
          const uint32_t at = atomicAdd(&met, 1u);
          if (at < kSampleList) {  // (always: sample_bins counted them)
            item_key[at] = t.key;
            item_index[at] = t.index;
          }
        }
      }
      sum = wave_sum64(sum);
      if (lane == 0) a.sub[(int64_t)r * a.subs + s0 / kSampleSub] = sum;
    }
  __syncthreads();
  if (met > 0) {  // this segment's part of the list, in any order
    if (tid == 0) ready = __hip_atomic_fetch_add(&a.ends[3 * r + 2], met, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    for (uint32_t i = tid; i < met && ready + i < kSampleList; i += 256)
      a.list[(int64_t)r * kSampleList + ready + i] = (uint64_t)item_key[i] << 32 | item_index[i];
  }
  if (!last_to_end(&a.ends[3 * r + 1], a.segs, &last)) return;

  const int listed = fits ? (int)in.listed : 0;
  for (int i = tid; i < listed; i += 256) {
    const uint64_t e = a.list[(int64_t)r * kSampleList + i];
    SampleItem t;
    item_of(float_of((uint32_t)(e >> 32)), (uint32_t)e, t);
    item_key[i] = t.key;
    item_index[i] = t.index;
    item_units[i] = t.heavy ? t.units : t.units | 1ull << 63;  // (units stay below 2^44)
    item_bin[i] = (uint16_t)t.bin;
  }
  for (int i = tid; i < a.subs; i += 256) sub[i] = fits ? a.sub[(int64_t)r * a.subs + i] : 0u;
  __syncthreads();
  // f(item) for this thread's share of the border's tokens
  auto each = [&](auto f) {
    if (fits) {
      for (int i = tid; i < listed; i += 256) {
        const uint64_t u = item_units[i];
        f(SampleItem{item_key[i], item_index[i], u & ~(1ull << 63), (int)item_bin[i], u >> 63 == 0});
      }
    } else {
      for (int i = 8 * tid; i < a.vocab; i += 2048) {
        float x[8];
        eight_logits<T>(row, i, a.vocab, x);
        for (int j = 0; j < 8; ++j) {
          SampleItem t;
          if (item_of(x[j], i + j, t) && at_border(t.bin)) f(t);
        }
      }
    }
  };
  // the sum of f(item) over them
  auto sum_of = [&](auto f) {
    uint64_t s = 0;
    each([&](const SampleItem& t) { s += f(t); });
    return block_sum64(s, four);
  };
  // the largest x with f(x), which holds at 0 and, where it holds, for everything smaller
  auto largest = [&](uint32_t lo, uint32_t hi, auto f) {  // f(lo) holds
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (f(mid)) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  // the bounds of the border's keys
  uint32_t key_lo = kNoIndex, key_hi = 0u;
  each([&](const SampleItem& t) {
    key_lo = t.key < key_lo ? t.key : key_lo;
    key_hi = t.key > key_hi ? t.key : key_hi;
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t x = (uint32_t)__shfl_xor((int)key_lo, o, 64), y = (uint32_t)__shfl_xor((int)key_hi, o, 64);
    key_lo = x < key_lo ? x : key_lo;
    key_hi = y > key_hi ? y : key_hi;
  }
  __syncthreads();
  if (lane == 0) four[w] = (uint64_t)key_hi << 32 | key_lo;
  __syncthreads();
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = (uint32_t)four[i], y = (uint32_t)(four[i] >> 32);
    key_lo = x < key_lo ? x : key_lo;
    key_hi = y > key_hi ? y : key_hi;
  }
  __syncthreads();

  // what stays: larger keys, and of those with this key the ones at smaller indices
  uint32_t key = 0u, below = kNoIndex;
  auto stays = [&](const SampleItem& t) { return t.key > key || (t.key == key && t.index < below); };
  // the first `n` of the tokens with key `x` that stay so far: the index behind them
  auto first_of = [&](uint32_t x, uint64_t n) {
    const auto equal = [&](const SampleItem& t) { return t.key == x && stays(t); };
    if (n >= sum_of([&](const SampleItem& t) { return (uint64_t)equal(t); })) return kNoIndex;
    // the last of them is the largest index in front of which there are fewer than n
    return 1u + largest(0u, (uint32_t)a.vocab, [&](uint32_t i) {
      return sum_of([&](const SampleItem& t) { return (uint64_t)(equal(t) && t.index < i); }) < n;
    });
  };
  uint64_t weight = in.all;
  if (bk >= 0) {
    const uint64_t want = in.k - in.count;  // tokens of bin bk that stay
    const uint32_t t = largest(key_lo, key_hi, [&](uint32_t x) {
      return sum_of([&](const SampleItem& i) { return (uint64_t)(i.bin == bk && i.key >= x); }) >= want;
    });
    const uint64_t over = sum_of([&](const SampleItem& i) { return (uint64_t)(i.bin == bk && i.key > t); });
    const uint32_t cut = first_of(t, want - over);
    key = t;
    below = cut;
    weight = in.weight + sum_of([&](const SampleItem& i) { return i.bin == bk && stays(i) ? i.units : 0ull; });
  }
  if (in.p < 1.0) {
    const uint64_t want = part(in.p, weight);
    const auto upto = [&](uint32_t x) {  // weight of the tokens with keys of at least x
      return in.before + sum_of([&](const SampleItem& i) { return i.bin >= plo && i.bin <= phi && i.key >= x && stays(i) ? i.units : 0ull; });
    };
    if (upto(key_lo) >= want) {
      const uint32_t t = largest(key_lo, key_hi, [&](uint32_t x) { return upto(x) >= want; });
      const uint64_t over = t == kNoIndex ? in.before : upto(t + 1u);
      SampleItem one;
      item_of(float_of(t), 0u, one);  // (t is the key of a token)
      const uint32_t cut = first_of(t, (want - over + one.units - 1) / one.units);
      below = t == key ? (cut < below ? cut : below) : cut;
      key = t;
    }
  }
  // the sums of 512 tokens each, with the border's
  if (fits) {
    each([&](const SampleItem& t) {
      if (stays(t) && t.heavy) atomicAdd(reinterpret_cast<unsigned long long*>(&sub[t.index / kSampleSub]), (unsigned long long)t.units);
    });
  } else {
    for (int s0 = kSampleSub * w; s0 < a.vocab; s0 += 4 * kSampleSub) {
      float x[8];
      const int i = s0 + 8 * lane;
      eight_logits<T>(row, i, a.vocab, x);
      uint64_t sum = 0;
      for (int j = 0; j < 8; ++j) {
        SampleItem t;
        if (item_of(x[j], i + j, t) && stays(t) && t.heavy) sum += t.units;
      }
      sum = wave_sum64(sum);
      if (lane == 0) sub[s0 / kSampleSub] = sum;
    }
  }
  __syncthreads();
  // which of them the random number falls into
  constexpr int kPer = kSampleSubs / 256;
  uint64_t mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mine[i] = kPer * tid + i < a.subs ? sub[kPer * tid + i] : 0u;
    sum += mine[i];
  }
  const uint64_t scan = wave_scan64(sum);
  if (lane == 63) four[w] = scan;
  __syncthreads();
  uint64_t before = scan - sum;
  for (int i = 0; i < w; ++i) before += four[i];
  const uint64_t all = four[0] + four[1] + four[2] + four[3];
  const double u = (double)a.u[r * a.u_s];
  const double aim = u > 0.0 ? floor(u * (double)all) : 0.0;  // (a NaN: 0)
  uint64_t target = aim < (double)all ? (uint64_t)aim : all - 1;
  if (target >= all) target = all - 1;  // (a sum that its double is larger than)
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (before <= target && target < before + mine[i]) {
      chosen = kPer * tid + i;
      left = target - before;
    }
    before += mine[i];
  }
  __syncthreads();
  if (w != 0) return;
  const int i0 = kSampleSub * chosen + 8 * lane;
  float x[8];
  eight_logits<T>(row, i0, a.vocab, x);
  uint64_t units[8];
  sum = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    SampleItem t;
    units[j] = item_of(x[j], i0 + j, t) && stays(t) && t.heavy ? t.units : 0u;
    sum += units[j];
  }
  uint64_t upto = wave_scan64(sum) - sum;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (upto <= left && left < upto + units[j]) a.out[r] = i0 + j;
    upto += units[j];
  }
}

// Tokens of a workgroup: enough workgroups for the card, where there are that many tokens.
static int sample_seg(int64_t rows, int64_t vocab) {
  int64_t seg = cdiv(cdiv(vocab * rows, 1024), 4 * kSampleSub) * 4 * kSampleSub;
  const int64_t whole = cdiv(vocab, 4 * kSampleSub) * 4 * kSampleSub;
  return (int)(seg < whole ? seg : whole);
}

struct SampleSpace {
  int64_t row, tops, weights, sub, list, counts, ends, lows, bytes;
};
static SampleSpace sample_space(int64_t rows, int64_t vocab) {
  const int64_t segs = cdiv(vocab, sample_seg(rows, vocab)), subs = cdiv(vocab, kSampleSub);
  SampleSpace s;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t x = at;
    at += (bytes + 15) & ~INT64_C(15);
    return x;
  };
  s.row = take(rows * sizeof(SampleRow));
  s.tops = take(rows * segs * 8);
  s.weights = take(rows * segs * kSampleBins * 8);
  s.sub = take(rows * subs * 8);
  s.list = take(rows * kSampleList * 8);
  s.counts = take(rows * segs * kSampleBins * 4);
  s.ends = take(rows * 3 * 4);
  s.lows = take(rows * segs * 4);
  s.bytes = at;
  return s;
}

template <typename T>
static int sample_launch(const SampleArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * a.segs));
  hipLaunchKernelGGL((sample_top<T>), grid, dim3(256), 0, s, a);
  if (const int rc = check_launch("sample_top")) return rc;
  hipLaunchKernelGGL((sample_bins<T>), grid, dim3(256), 0, s, a);
  if (const int rc = check_launch("sample_bins")) return rc;
  hipLaunchKernelGGL((sample_pick<T>), grid, dim3(256), 0, s, a);
  return check_launch("sample_pick");
}

}  // namespace biops

using namespace biops;

extern "C" int64_t biops_sample_workspace_size(int64_t rows, int64_t vocab) {
  if (rows < 0 || vocab < 1 || vocab > kSampleMost || rows > 65536) return -1;
  return rows == 0 ? 0 : sample_space(rows, vocab).bytes;
}

extern "C" int biops_sample(int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const float* u, int64_t u_s,
                            const float* temperature, int64_t t_s, double t0, const void* top_k, int k64, int64_t k_s, int64_t k0,
                            const float* top_p, int64_t p_s, double p0, const float* min_p, int64_t m_s, double m0, int64_t* out,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  if (!is_float_dtype(dtype)) return fail(BIOPS_ERR_DTYPE, "biops_sample: unsupported dtype %d", dtype);
  if (rows < 0 || rows > 65536 || vocab < 1 || vocab > kSampleMost)
    return fail(BIOPS_ERR_ARG, "biops_sample: rows of 1 to %d tokens, at most 65536 rows", kSampleMost);
  if (rows == 0) return BIOPS_OK;
  if (!logits || !u || !out) return fail(BIOPS_ERR_ARG, "biops_sample: null pointer");
  const SampleSpace x = sample_space(rows, vocab);
  if (!workspace || workspace_bytes < x.bytes)
    return fail(BIOPS_ERR_SIZE, "biops_sample: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)x.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BIOPS_ERR_LAYOUT, "biops_sample: workspace not 16-byte aligned");
  SampleArgs a;
  a.logits = static_cast<const char*>(logits), a.ld = dtype_bytes(dtype) * ld;
  a.u = u, a.temperature = temperature, a.top_p = top_p, a.min_p = min_p, a.top_k = top_k;
  a.u_s = u_s, a.t_s = t_s, a.k_s = k_s, a.p_s = p_s, a.m_s = m_s;
  a.t0 = t0, a.p0 = p0, a.m0 = m0, a.k0 = k0, a.k64 = k64 != 0;
  a.out = out, a.rows = (int)rows, a.vocab = (int)vocab;
  a.seg = sample_seg(rows, vocab), a.segs = (int)cdiv(vocab, a.seg), a.subs = (int)cdiv(vocab, kSampleSub);
  char* const base = static_cast<char*>(workspace);
  a.row = reinterpret_cast<SampleRow*>(base + x.row);
  a.tops = reinterpret_cast<uint64_t*>(base + x.tops), a.weights = reinterpret_cast<uint64_t*>(base + x.weights);
  a.sub = reinterpret_cast<uint64_t*>(base + x.sub), a.list = reinterpret_cast<uint64_t*>(base + x.list);
  a.counts = reinterpret_cast<uint32_t*>(base + x.counts), a.ends = reinterpret_cast<uint32_t*>(base + x.ends);
  a.lows = reinterpret_cast<float*>(base + x.lows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  BIOPS_DISPATCH_FLOAT(dtype, return sample_launch<T>(a, s));
  return BIOPS_OK;
}

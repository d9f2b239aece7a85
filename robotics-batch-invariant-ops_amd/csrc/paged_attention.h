// What the attentions of one new token over pages share: the keys a sequence sees, the chunks they are cut into, and the
// join of the chunks' results.
#pragma once

#include <type_traits>

#include "gemm_core.h"
#include "rowops.h"
#include "scores.h"

namespace biops {

constexpr int kPagedKeys = 128;    // keys of the shortest chunk: a tile of 32 for each of four wavefronts
constexpr int kPagedChunks = 64;   // most chunks of a sequence
constexpr int kPagedCols = 16;     // query heads of a workgroup
// Powers of two that fp16 weights are larger by (up to half of the type's range, where they may be 2^8): those down to 2^-32 of the
// largest count (2^-25 without: of 128 keys beside one of weight 1 whose value is 0, 31 of weight e^-15 were off by 2.6 %, and
// at e^-18 gone).
template <typename T> constexpr float kPagedUp = std::is_same<T, f16_t>::value ? 7.f : 0.f;

struct PagedArgs {
  const char *q, *kc, *vc;
  char* out;
  float *part, *ml;                       // chunk results: [row][chunk][dv], [row][chunk][2]
  const void *table, *lengths;
  int* flag;
  int64_t qB, qH, kP, kS, kH, vP, vS, vH;  // byte strides
  int64_t tB, tW, lB;                      // element strides of the page table and the lengths
  uint32_t batch, hkv, group, zs;          // zs: workgroups per key/value head (16 query heads each)
  uint32_t page_size;
  int64_t pages;
  int limit;                               // longest length that the table (and the caller) allow
  uint32_t first, rows;                    // first workgroup of a launch; batch * hkv * zs
  int d, dv, chunks;                       // chunks: most chunks of a sequence
  int window, sinks;                       // window 0: all
  int table64, lengths64;
  int negate, zero;                        // the scale is negative, or 0 (score_scale)
  float scale;                             // c > 0
};

struct PagedSpan {
  int n;          // visible keys
  int ns, shift;  // key of v: v < ns ? v : v + shift
  int chunk;      // keys per chunk
  int chunks;
  bool bad;
};

// Keys per chunk, by the number of visible keys alone.  Short sequences need their chunks for units to run on, long
// ones have enough of them, and every chunk starts with three reads that wait for one another and ends with a result
// to be joined.  us by chunk size (128 / 256 / 512): 16/4 heads of 128, one sequence of 2047 keys 10.4 / 12.5 / 13,
// 64 of 3920 keys 130 / 120 / 111; 32/8 heads, 128 sequences of 1024 keys 138 / 123 / 117 (what one sequence of that
// length gains weighs more: in a batch of one every layer of every token pays it).
__host__ __device__ __forceinline__ int paged_chunk(int n) {
  if (n <= 2048) return kPagedKeys;
  if (n <= 4096) return 2 * kPagedKeys;
  constexpr int most = 4 * kPagedKeys * kPagedChunks;
  return 4 * kPagedKeys * (n <= most ? 1 : (n - 1) / most + 1);
}

// Length of sequence b, -1 where it is outside of what the table allows.
__device__ __forceinline__ int paged_length(const PagedArgs& a, int64_t b) {
  const int64_t len = a.lengths64 ? reinterpret_cast<const int64_t*>(a.lengths)[b * a.lB]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.lengths)[b * a.lB];
  return len < 0 || len > a.limit ? -1 : (int)len;
}

__device__ __forceinline__ PagedSpan paged_span(const PagedArgs& a, int len) {
  PagedSpan s;
  s.bad = len < 0;
  const int l = s.bad ? 0 : len;
  const int start = a.window > 0 && l > a.window ? l - a.window : 0;
  s.ns = a.sinks < start ? a.sinks : start;
  s.shift = start - s.ns;
  s.n = s.ns + l - start;
  s.chunk = paged_chunk(s.n);
  // (a power of two up to the length from which a sequence has all its chunks: a division is 20 instructions)
  s.chunks = s.n <= 4 * kPagedKeys * kPagedChunks ? (s.n + s.chunk - 1) >> (31 - __builtin_clz((uint32_t)s.chunk)) : (s.n - 1) / s.chunk + 1;
  return s;
}

// Work item `it` of a batch of up to 128 sequences: chunk c of sequence b, all chunks of the first sequence, then of the
// next.  Counting them here, two sequences a lane, leaves no idle workgroups between those with work (64 sequences of 250
// to 16384 keys: 142 us with a workgroup for every chunk that the longest sequence could have, 113 so).
constexpr uint32_t kPagedListed = 128;
__device__ __forceinline__ bool paged_find(const PagedArgs& a, int it, int lane, uint32_t& b, int& c, int& length) {
  const uint32_t first = 2 * lane;
  const int len0 = first < a.batch ? paged_length(a, first) : 0;
  const int len1 = first + 1 < a.batch ? paged_length(a, first + 1) : 0;
  const int one = paged_span(a, len0).chunks, both = one + paged_span(a, len1).chunks;
  int upto = both;
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8: sums in rows of 16 lanes
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x142, 0xa, 0xf, false);  // row_bcast:15, 31: over the rows
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x143, 0xc, 0xf, false);
  const uint64_t hit = __ballot(upto > it);
  if (hit == 0) return false;
  const int f = __builtin_ctzll(hit);
  c = it - (__builtin_amdgcn_readlane(upto, f) - __builtin_amdgcn_readlane(both, f));
  const int in_first = __builtin_amdgcn_readlane(one, f);
  const bool second = c >= in_first;
  b = 2 * f + second;
  if (second) c -= in_first;
  length = second ? __builtin_amdgcn_readlane(len1, f) : __builtin_amdgcn_readlane(len0, f);
  return true;
}

template <typename T>
__device__ __forceinline__ void mfma16(f32x4_t& acc, const u32x4_t& a, const u32x4_t& b) {
  if constexpr (std::is_same<T, bf16_t>::value)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
  else if constexpr (std::is_same<T, f16_t>::value)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), acc, 0, 0, 0);
  else
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), acc, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float x, float y) {
  if constexpr (std::is_same<T, bf16_t>::value) return f32x2_to_bf16x2_bits(x, y);
  else return f32x2_to_f16x2_bits(x, y);
}

// The end of a chunk's workgroup: the four wavefronts' results as means and what they count for, joined in order, and the
// output row or the chunk's place in the workspace.  Query m16's largest product m and sum l (of this lane's keys), acc[t][i]
// the sums of column 16 W n + W (4 q4 + i) + t % W (n = t / W), all less `down` powers of two.
template <typename T, int DVP, int W>
__device__ __forceinline__ void paged_finish(const PagedArgs& a, char* smem, int* bad_page, float m, float l, float down, bool bad,
                                             const f32x4_t (&acc)[DVP / 16], uint32_t b, int64_t h0, int c, int cols) {
  constexpr int NB = DVP / (16 * W);
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int m16 = lane & 15, q4 = lane >> 4;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (bad) *bad_page = 1;

  // the four wavefronts' results: means and what they count for, joined in order
  float* const os = reinterpret_cast<float*>(smem);
  float* const mls = os + 4 * cols * DVP;
  if (m16 < cols) {
    if (q4 == 0) {
      mls[2 * (w * cols + m16)] = m;
      mls[2 * (w * cols + m16) + 1] = l * __builtin_amdgcn_exp2f(down);
    }
    float* o = os + (w * cols + m16) * DVP;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < W; t += 4)
          *reinterpret_cast<f32x4_t*>(o + 16 * W * n + W * (4 * q4 + i) + t) =
              f32x4_t{acc[W * n + t][i], acc[W * n + t + 1][i], acc[W * n + t + 2][i], acc[W * n + t + 3][i]} * inv;
  }
  __syncthreads();
  const bool void_ = *bad_page != 0;
  if (void_ && tid == 0) *a.flag = 1;
  const int64_t heads = (int64_t)a.hkv * a.group;
  const int pieces = a.dv >> 2;
  for (int i = tid; i < cols * pieces; i += 256) {
    const int col = i / pieces, e = 4 * (i - col * pieces);
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < 4; ++x) M = fmaxf(M, mls[2 * (x * cols + col)]);
    const float base = M == -INFINITY ? 0.f : M;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    float f[4], sum = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f[x] = mls[2 * (x * cols + col) + 1] * __builtin_amdgcn_exp2f((mls[2 * (x * cols + col)] - base) * a.scale);
      sum += f[x];
    }
    const float share = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int x = 0; x < 4; ++x) o += *reinterpret_cast<const f32x4_t*>(os + (x * cols + col) * DVP + e) * (f[x] * share);
    const int64_t row = b * heads + h0 + col;
    if (a.chunks == 1) {
      T* dst = reinterpret_cast<T*>(a.out) + row * a.dv + e;
#pragma unroll
      for (int x = 0; x < 4; ++x) Num<T>::store(dst + x, void_ ? 0.f : o[x]);
    } else {
      const int64_t at = row * a.chunks + c;
      *reinterpret_cast<f32x4_t*>(a.part + at * a.dv + e) = o;
      if (e == 0) {
        a.ml[2 * at] = M;
        a.ml[2 * at + 1] = void_ ? -1.f : sum;
      }
    }
  }
}

// Joins the chunks of one output row per workgroup.  Thread (split, piece) adds chunks split, split + S,
// ... for four columns; the splits are then added in order.
template <typename T>
static __global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  __shared__ float top, total;
  __shared__ int void_row;
  __shared__ __attribute__((aligned(16))) f32x4_t so[256];
  const int tid = threadIdx.x;
  const int64_t row = a.first + blockIdx.x;
  const float* ml = a.ml + 2 * row * a.chunks;
  const float* part = a.part + row * a.chunks * a.dv;
  const int pieces = a.dv >> 2, splits = 256 / pieces;
  const int piece = tid % pieces, split = tid / pieces;
  // The first reads do not wait for the length: their places exist, whether a chunk is there or not.
  float m0 = -INFINITY, l0 = 0.f, ms = 0.f, ls = 0.f;
  f32x4_t os = {0.f, 0.f, 0.f, 0.f};
  if (tid < a.chunks) {
    m0 = ml[2 * tid];
    l0 = ml[2 * tid + 1];
  }
  if (split < splits && split < a.chunks) {
    ms = ml[2 * split];
    ls = ml[2 * split + 1];
    os = *reinterpret_cast<const f32x4_t*>(part + (int64_t)split * a.dv + 4 * piece);
  }
  const PagedSpan span = paged_span(a, paged_length(a, (uint32_t)row / (a.hkv * a.group)));
  T* dst = reinterpret_cast<T*>(a.out) + row * a.dv;
  if (span.bad && tid == 0) *a.flag = 1;
  // (a sequence has at most 64 chunks: the first wavefront sees them all)
  static_assert(kPagedChunks <= 64, "one wavefront holds all chunks' maxima");
  if (tid < 64) {
    const bool there = tid < span.chunks;
    const float mx = wave_max(there ? m0 : -INFINITY);
    const bool bad = __any(there && l0 == -1.f);
    const float all = wave_sum(there ? l0 * __builtin_amdgcn_exp2f((m0 - (mx == -INFINITY ? 0.f : mx)) * a.scale) : 0.f);
    if (tid == 0) {
      top = mx == -INFINITY ? 0.f : mx;
      total = all;
      void_row = bad || all == 0.f;
    }
  }
  __syncthreads();
  const float base = top, sum = total;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  if (split < splits)
    for (int c = split; c < span.chunks; c += splits) {
      if (c != split) {
        ms = ml[2 * c];
        ls = ml[2 * c + 1];
        os = *reinterpret_cast<const f32x4_t*>(part + (int64_t)c * a.dv + 4 * piece);
      }
      o += os * (ls * __builtin_amdgcn_exp2f((ms - base) * a.scale) / sum);  // (of one chunk 1 exactly)
    }
  so[tid] = o;
  __syncthreads();
  if (split == 0) {
    const int filled = span.chunks < splits ? span.chunks : splits;
    for (int s = 1; s < filled; ++s) o += so[s * pieces + piece];
#pragma unroll
    for (int x = 0; x < 4; ++x) Num<T>::store(dst + 4 * piece + x, void_row ? 0.f : o[x]);
  }
}

// The join of a launch's output rows, where a sequence can have several chunks.
template <typename T>
static int paged_join(PagedArgs& a, hipStream_t s) {
  constexpr uint32_t most = 1 << 22;  // a launch has less than 2^32 threads
  const uint32_t joins = a.batch * a.hkv * a.group;
  for (a.first = 0; a.chunks > 1 && a.first < joins; a.first += most) {
    const uint32_t n = joins - a.first < most ? joins - a.first : most;
    hipLaunchKernelGGL((paged_join_kernel<T>), dim3(n), dim3(256), 0, s, a);
    const int rc = check_launch("paged_join_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}

// Longest length taken: the table's pages, the caller's bound, and 31-bit positions.
static inline int64_t paged_limit(int64_t width, int64_t page_size, int64_t max_length) {
  const int64_t most = INT64_C(0x7fffffff);
  int64_t limit = page_size > 0 && width > most / page_size ? most : width * page_size;
  if (max_length >= 0 && max_length < limit) limit = max_length;
  return limit;
}
// Most chunks that a sequence of up to `limit` keys can have: the count grows with the visible keys between the sizes
// at which chunks grow.
static inline int paged_chunks(int64_t limit, int64_t window, int64_t sinks) {
  int64_t n = limit;
  if (window > 0 && window < limit && sinks < limit - window) n = window + sinks;
  int most = 1;
  for (const int64_t x : {INT64_C(2048), INT64_C(4096), n}) {
    const int64_t m = x < n ? x : n;
    const int64_t c = m > 0 ? (m - 1) / paged_chunk((int)m) + 1 : 1;
    if (c > most) most = (int)c;
  }
  // past the last size the count saw-tooths below its bound
  return n > (int64_t)4 * kPagedKeys * kPagedChunks ? kPagedChunks : most;
}

}  // namespace biops

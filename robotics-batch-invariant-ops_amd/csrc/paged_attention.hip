// Attention of one new token per sequence over a cache in pages, with an optional sliding window and
// first tokens (sinks) that stay visible.
//
// Sequence b has L keys in its pages; its query is the token at L - 1.  It sees key j where j < sinks
// or j >= L - window.  The visible keys are counted through: v = 0 .. n - 1, the sinks in front of the
// window first, so that nothing else is loaded or looked up.  They are cut into chunks, a workgroup takes
// a chunk of one key/value head for all the query heads that share it, and a second kernel joins the
// chunks in their order (none where no sequence can have more than one):
//   chunk:  m = max s_v, l = sum exp2(c (s_v - m)), o = sum exp2(c (s_v - m)) V_v / l,  s_v = q.k_v, c = scale log2 e
//   join:   M = max m_c, L_c = exp2(c (m_c - M)) l_c, o = sum_c (L_c / sum L) o_c
// The difference is taken before the product with c: it is exact next to the maximum however large the scores are, where
// a fused c s_v - round(c m) would leave the rounding of c m in every weight, powers of two that overflow from 2^31 on.
// Batch invariance: the chunks follow from n alone, so a sequence's bits are the same in every batch.
//
// What bounds it is the stream of keys and values, read once: about 4 G operations per 2-byte element (G
// query heads per key head), far below what the matrix cores do, so these run mostly empty (16 columns
// for G queries).  Neither operand passes through LDS:
//   S^T = K Q^T by 16x16 MFMAs: lane (m = lane % 16, q = lane / 16) loads 16-byte pieces of key row m.
//     Row m of score block i (i = 0, 1 of a tile of 32 keys) is key 8 (m / 4) + 4 i + m % 4, so that a lane
//     ends up with the scores of keys 8q .. 8q + 7 of query m;
//   O^T = V^T P^T: those eight are the lane's part of the B operand as they stand.  For A the lane loads W
//     elements (16 bytes; 8 with 64-wide heads) of value rows 8q .. 8q + 7 at column W m -- whole
//     rows, contiguous over the lanes -- and turns its own 8 x W block with byte permutes: row m of output
//     block t is column W m + t.
// Parts are joined as means, which stay in the range of their values; a wavefront whose own sum has left it goes through its
// keys once more, with weights so much smaller that as many of the largest values stay in it (always so, small values would
// lose bits).  Sums of fp16 values cannot get there.
// 16-bit weights go in as a rounded part and the rounded rest (two MFMAs), which leaves an error of
// 2^-16 (bf16) instead of 2^-8 where the matrix cores have the time.
//
// bf16, 16/4 heads of 128, 64 sequences of 250 to 16384 keys: 114 us, 4.5 TB/s (a copy of as many bytes: 103), and 5 for
// the join; one sequence of 2047 keys 7 and 4; fp16, 8/2 heads of 64, 100 sequences under a window of 1024: 11.6 and 4.
//
// Slots behind the end of a sequence may hold anything: keys of the last tile past the end are read
// from the last key's row, their scores replaced by -inf and their values by zeros.
#include <type_traits>

#include "gemm_core.h"
#include "rowops.h"
#include "scores.h"

namespace biops {

constexpr int kPagedKeys = 128;    // keys of the shortest chunk: a tile of 32 for each of four wavefronts
constexpr int kPagedChunks = 64;   // most chunks of a sequence
constexpr int kPagedCols = 16;     // query heads of a workgroup

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
  s.chunks = s.n > 0 ? (s.n - 1) / s.chunk + 1 : 0;
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
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o, 64);
    if (lane >= o) upto += x;
  }
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

// Wavefronts per SIMD that registers are given out for.
template <typename T, int DP, int DVP>
constexpr int paged_waves() {
  constexpr int wide = (DP > DVP ? DP : DVP) * (sizeof(T) / 2);
  return wide <= 64 ? 4 : (wide <= 128 ? 3 : (wide <= 256 ? 2 : 1));
}

template <typename T, int DP, int DVP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(paged_waves<T, DP, DVP>(), paged_waves<T, DP, DVP>())))
void paged_chunk_kernel(PagedArgs a) {
  constexpr int E = sizeof(T), VEC = 16 / E;
  constexpr int KW = 4 * VEC, KS = DP / KW;             // elements and number of the score steps
  constexpr int W = E == 2 && DVP <= 64 ? 4 : VEC;      // elements of a value load
  constexpr int NB = DVP / (16 * W), NT = NB * W;       // value blocks of a row; 16-column output blocks
  constexpr int VD = W * E / 4;                         // dwords of a value load
  extern __shared__ __attribute__((aligned(16))) char smem[];  // [4][cols][DVP] O, then [4][cols][2] m, l
  __shared__ __attribute__((aligned(16))) int64_t offs[4][2][32];
  __shared__ int bad_page;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int m16 = lane & 15, q4 = lane >> 4;
  const u32x4_t zero4 = {0u, 0u, 0u, 0u};
  const int64_t heads = (int64_t)a.hkv * a.group;

  uint32_t r = a.first + blockIdx.x;
  const uint32_t z = r % a.zs;
  r /= a.zs;
  const uint32_t hk = r % a.hkv;
  uint32_t b = r / a.hkv;
  int c = 0, length;
  if (a.chunks == 1) {
    length = paged_length(a, b);
  } else if (a.batch <= kPagedListed) {
    if (!paged_find(a, (int)b, lane, b, c, length)) return;
  } else {  // first chunks of all sequences, then second ones: what is idle comes last
    c = (int)(b / a.batch);
    b -= c * a.batch;
    length = paged_length(a, b);
  }
  const PagedSpan span = paged_span(a, length);
  if (a.chunks > 1 && c >= span.chunks) return;
  const int cols = a.group - z * kPagedCols < kPagedCols ? (int)(a.group - z * kPagedCols) : kPagedCols;
  const int64_t h0 = hk * a.group + z * kPagedCols;
  if (span.chunks == 0) {  // (one chunk at most, and no join) a row that sees nothing
    if (span.bad) *a.flag = 1;
    for (int i = tid; i < cols * a.dv; i += 256)
      Num<T>::store(reinterpret_cast<T*>(a.out) + (b * heads + h0) * a.dv + i, 0.f);
    return;
  }
  if (tid == 0) bad_page = 0;
  const int v0 = c * span.chunk;
  const int nkeys = span.n - v0 < span.chunk ? span.n - v0 : span.chunk;
  const int tiles = (nkeys + 31) >> 5;

  // queries (B operand): lane holds query column m16, elements KW s + VEC q4 ..
  u32x4_t qf[KS];
  {
    const char* qr = a.q + b * a.qB + (h0 + (m16 < cols ? m16 : 0)) * a.qH;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = KW * s + VEC * q4;
      qf[s] = m16 < cols && d0 < a.d ? load_16(qr + E * d0) : zero4;
      if (a.negate | a.zero) qf[s] = score_query<T>(qf[s], a.negate, a.zero);
    }
  }
  __syncthreads();  // bad_page is clear

  // byte offset of key `lane % 32` of a tile in the key cache (lanes 0-31) or the value cache
  bool bad = false;
  auto lookup = [&](int tile) -> int64_t {
    int i = 32 * tile + (lane & 31);
    if (i >= nkeys) i = nkeys - 1;
    const int v = v0 + i;
    const uint32_t key = (uint32_t)(v < span.ns ? v : v + span.shift);
    const uint32_t page = key / a.page_size, at = key - page * a.page_size;
    const int64_t e = b * a.tB + page * a.tW;
    int64_t id = a.table64 ? reinterpret_cast<const int64_t*>(a.table)[e]
                           : (int64_t) reinterpret_cast<const int32_t*>(a.table)[e];
    if (id < 0 || id >= a.pages) {
      bad = true;
      id = 0;
    }
    return lane < 32 ? id * a.kP + at * a.kS : id * a.vP + at * a.vS;
  };

  const char* const kb = a.kc + hk * a.kH;
  const char* const vb = a.vc + hk * a.vH;
  // of query m16: largest product so far, the same or 0 where that is -inf, sum (of this lane's keys)
  float m, from, l;
  f32x4_t acc[NT];
  float down = 0.f;  // powers of two that are off the weights
  for (;;) {
    m = -INFINITY, from = 0.f, l = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    int64_t off = w < tiles ? lookup(w) : 0;
    for (int tile = w; tile < tiles; tile += 4) {
      offs[w][lane >> 5][lane & 31] = off;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      u32x4_t kf[2][KS];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const char* p = kb + offs[w][0][8 * (m16 >> 2) + 4 * i + (m16 & 3)];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int d0 = KW * s + VEC * q4;
          kf[i][s] = d0 < a.d ? load_16(p + E * d0) : zero4;
        }
      }
      uint32_t vf[NB][8][VD];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const char* p = vb + offs[w][1][8 * q4 + j];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int e0 = 16 * W * n + W * m16;
          if constexpr (VD == 4) {
            const u32x4_t x = e0 < a.dv ? load_16(p + E * e0) : zero4;
#pragma unroll
            for (int i = 0; i < 4; ++i) vf[n][j][i] = x[i];
          } else {
            const u32x2_t x = e0 < a.dv ? *reinterpret_cast<const u32x2_any_t*>(p + E * e0) : u32x2_t{0u, 0u};
            vf[n][j][0] = x[0];
            vf[n][j][1] = x[1];
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (tile + 4 < tiles) off = lookup(tile + 4);

      f32x4_t sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) mfma16<T>(sc[i], kf[i][s], qf[s]);
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = sc[j >> 2][j & 3];
      const int left = nkeys - 32 * tile;
      if (left < 32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = 8 * q4 + j < left;
          p[j] = in ? p[j] : -INFINITY;
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < VD; ++i) vf[n][j][i] = in ? vf[n][j][i] : 0u;
        }
      }
      float mx = p[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, p[j]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float corr = mx > m ? __builtin_amdgcn_exp2f((m - mn) * a.scale) : 1.f;
        l *= corr;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] *= corr;
        m = mn;
        from = mn == -INFINITY ? 0.f : mn;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[j] - from, a.scale, -down));
        l += p[j];
      }
      if constexpr (E == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int t = 0; t < W; ++t)
              acc[W * n + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[n][j][t]), p[j], acc[W * n + t], 0, 0, 0);
      } else {
        u32x4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[i] = pack_pair<T>(p[2 * i], p[2 * i + 1]);
          lo[i] = pack_pair<T>(p[2 * i] - Num<T>::from_bits(hi[i] & 0xffffu), p[2 * i + 1] - Num<T>::from_bits(hi[i] >> 16));
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int t = 0; t < W; ++t) {
            u32x4_t va;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              va[i] = __builtin_amdgcn_perm(vf[n][2 * i + 1][t >> 1], vf[n][2 * i][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            mfma16<T>(acc[W * n + t], va, hi);
            mfma16<T>(acc[W * n + t], va, lo);
          }
      }
    }
    if constexpr (std::is_same<T, f16_t>::value) break;
    float odd = 0.f;  // NaN where a sum of the query is not finite
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) odd = __builtin_fmaf(acc[t][i], 0.f, odd);
    odd += __shfl_xor(odd, 16, 64);
    odd += __shfl_xor(odd, 32, 64);
    const bool past = odd != 0.f && down == 0.f && m16 < cols;
    if (!__any(past)) break;
    if (past) down = (float)(32 - __builtin_clz((uint32_t)span.chunk / 4));  // (a wavefront has a quarter of the chunk's keys)
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (bad) bad_page = 1;

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
  const bool void_ = bad_page != 0;
  if (void_ && tid == 0) *a.flag = 1;
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
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
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

template <typename T, int DP, int DVP>
static int paged_launch(PagedArgs a, hipStream_t s) {
  const unsigned cols = a.group < kPagedCols ? a.group : kPagedCols;
  const unsigned lds = (unsigned)(4 * cols * (DVP + 2) * sizeof(float));
  constexpr uint32_t most = 1 << 22;  // a launch has less than 2^32 threads
  const uint32_t total = a.rows * a.chunks, joins = a.batch * a.hkv * a.group;
  for (a.first = 0; a.first < total; a.first += most) {
    const uint32_t n = total - a.first < most ? total - a.first : most;
    hipLaunchKernelGGL((paged_chunk_kernel<T, DP, DVP>), dim3(n), dim3(256), lds, s, a);
    const int rc = check_launch("paged_chunk_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  for (a.first = 0; a.chunks > 1 && a.first < joins; a.first += most) {
    const uint32_t n = joins - a.first < most ? joins - a.first : most;
    hipLaunchKernelGGL((paged_join_kernel<T>), dim3(n), dim3(256), 0, s, a);
    const int rc = check_launch("paged_join_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}
template <typename T, int DP>
static int paged_launch_dv(const PagedArgs& a, hipStream_t s) {
  if (a.dv <= 64) return paged_launch<T, DP, 64>(a, s);
  if (a.dv <= 128) return paged_launch<T, DP, 128>(a, s);
  return paged_launch<T, DP, 256>(a, s);
}
template <typename T>
static int paged_launch_d(const PagedArgs& a, hipStream_t s) {
  if (a.d <= 64) return paged_launch_dv<T, 64>(a, s);
  if (a.d <= 128) return paged_launch_dv<T, 128>(a, s);
  return paged_launch_dv<T, 256>(a, s);
}

// Longest length taken: the table's pages, the caller's bound, and 31-bit positions.
static int64_t paged_limit(int64_t width, int64_t page_size, int64_t max_length) {
  const int64_t most = INT64_C(0x7fffffff);
  int64_t limit = page_size > 0 && width > most / page_size ? most : width * page_size;
  if (max_length >= 0 && max_length < limit) limit = max_length;
  return limit;
}
// Most chunks that a sequence of up to `limit` keys can have: the count grows with the visible keys between the sizes
// at which chunks grow.
static int paged_chunks(int64_t limit, int64_t window, int64_t sinks) {
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

using namespace biops;

extern "C" int64_t biops_paged_attention_workspace_size(int64_t batch, int64_t hq, int64_t dv, int64_t width,
                                                        int64_t page_size, int64_t max_length, int64_t window,
                                                        int64_t sinks) {
  if (batch < 0 || hq < 0 || dv < 0 || dv > 256 || width < 0 || page_size < 0 || window < 0 || sinks < 0) return -1;
  const int chunks = paged_chunks(paged_limit(width, page_size, max_length), window, sinks);
  if (chunks == 1 || batch == 0 || hq == 0) return 0;
  if (hq > (INT64_C(1) << 30) / kPagedChunks / batch) return -1;
  return batch * hq * chunks * (dv + 2) * (int64_t)sizeof(float);
}

extern "C" int biops_paged_attention(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t dv,
                                     const void* q, int64_t sqB, int64_t sqH, const void* kc, int64_t skP, int64_t skS,
                                     int64_t skH, const void* vc, int64_t svP, int64_t svS, int64_t svH, int64_t pages,
                                     int64_t page_size, const void* table, int table64, int64_t stB, int64_t stW,
                                     int64_t width, const void* lengths, int lengths64, int64_t slB, int64_t max_length,
                                     int64_t window, int64_t sinks, float scale, void* out, int* flag, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  const int elt = is_float_dtype(dtype) ? dtype_bytes(dtype) : 0;
  if (elt == 0) return fail(BIOPS_ERR_DTYPE, "biops_paged_attention: unsupported dtype %d", dtype);
  if (batch < 0 || hq < 0 || hkv <= 0 || hq % hkv != 0) return fail(BIOPS_ERR_ARG, "biops_paged_attention: bad batch or heads");
  const int vec = 16 / elt;
  if (d < vec || d > 256 || d % vec || dv < vec || dv > 256 || dv % vec)
    return fail(BIOPS_ERR_ARG, "biops_paged_attention: head sizes are multiples of %d up to 256", vec);
  if (pages <= 0 || page_size <= 0 || width < 0 || page_size > INT64_C(0x7fffffff))
    return fail(BIOPS_ERR_ARG, "biops_paged_attention: a cache without pages");
  if (window < 0 || sinks < 0) return fail(BIOPS_ERR_ARG, "biops_paged_attention: negative window");
  if (!(scale - scale == 0.f)) return fail(BIOPS_ERR_ARG, "biops_paged_attention: scale is not finite");
  if (batch == 0 || hq == 0) return BIOPS_OK;
  if (!q || !kc || !vc || !lengths || !out || !flag || (width > 0 && !table))
    return fail(BIOPS_ERR_ARG, "biops_paged_attention: null pointer");
  // counted in 32 bits: workgroups and output rows
  if (hq > (INT64_C(1) << 30) / kPagedChunks / batch) return fail(BIOPS_ERR_ARG, "biops_paged_attention: more than 2^24 rows");
  PagedArgs a;
  const int64_t limit = paged_limit(width, page_size, max_length), all = INT64_C(0x7fffffff);
  a.limit = (int)limit;
  a.chunks = paged_chunks(limit, window, sinks);
  a.batch = (uint32_t)batch, a.hkv = (uint32_t)hkv, a.group = (uint32_t)(hq / hkv);
  a.zs = (a.group + kPagedCols - 1) / kPagedCols;
  a.rows = a.batch * a.hkv * a.zs;
  const int64_t rows = batch * hq * a.chunks;
  if (a.chunks > 1) {
    const int64_t need = rows * (dv + 2) * (int64_t)sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(BIOPS_ERR_SIZE, "biops_paged_attention: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BIOPS_ERR_LAYOUT, "biops_paged_attention: workspace not 16-byte aligned");
  }
  a.part = static_cast<float*>(workspace);
  a.ml = a.part + rows * dv;
  a.q = static_cast<const char*>(q), a.kc = static_cast<const char*>(kc), a.vc = static_cast<const char*>(vc);
  a.out = static_cast<char*>(out);
  a.table = table, a.lengths = lengths, a.flag = flag;
  a.qB = elt * sqB, a.qH = elt * sqH;
  a.kP = elt * skP, a.kS = elt * skS, a.kH = elt * skH;
  a.vP = elt * svP, a.vS = elt * svS, a.vH = elt * svH;
  a.tB = stB, a.tW = stW, a.lB = slB;
  a.pages = pages, a.page_size = (uint32_t)page_size;
  a.d = (int)d, a.dv = (int)dv;
  a.window = (int)(window < all ? window : all), a.sinks = (int)(sinks < all ? sinks : all);
  a.table64 = table64 != 0, a.lengths64 = lengths64 != 0;
  a.scale = score_scale(scale, &a.negate, &a.zero);
  hipStream_t s = static_cast<hipStream_t>(stream);
  BIOPS_DISPATCH_FLOAT(dtype, return paged_launch_d<T>(a, s));
  return BIOPS_OK;
}

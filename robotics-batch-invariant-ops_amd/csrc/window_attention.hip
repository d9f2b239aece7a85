// Attention under a sliding window with a few first tokens (sinks) that stay visible: prompts and chunks
// of new tokens, dense [batch, heads, tokens, dim] or packed by sequence.
//
// Query r of a sequence (lq queries, lk keys) is the token at p = lk - lq + r and sees the keys j <= p
// with p - j < window or j < sinks:  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q.k_j.
//
// A workgroup's wavefronts own 32 query rows each, of one head or of several that share a key/value head
// (window_launch_rows has the variants and what they measured), and pass once over the keys that any of
// them sees, counted through from 0: the sinks in front of the first row's window, then everything up to the last
// row.  So the sinks share the first block with the window's first keys, and work grows with the window, not with the
// sequence.  Blocks of 64 keys go straight from memory to LDS; running maximum m and sum l per row, O rescaled when a
// maximum has grown enough.
//
// Register layout: S^T = K Q^T (K as the A operand of 32x32 MFMAs) leaves lane L with query row L % 32 and
// keys 8j + 4(L/32) + i of a 32-key block, which is the B operand of O^T = V^T P^T with the same key order
// in V; so weights go from accumulators to the next MFMA without LDS, and a row's maximum, sum and rescale
// stay in its lane (one exchange between the two lanes of a row).  16-bit V fragments come from LDS by
// the transposing read.  16-bit weights are rounded once to the type for the product (half a step, as the
// output's own rounding); statistics and sums are 32-bit.
//
// A masked key never reaches a row, to the bit.  Its scores are replaced, not added to, and 0 times its values adds nothing
// unless one of them is not finite: a row whose sum is finite and whose output is not is computed again, in the same blocks
// and order over values whose infinities and NaN are zeros (mode 1), and those that the row sees are then set in its output
// (window_mark).  If it still is not finite, its sum passed float's range where the mean does not: once more with smaller
// weights (mode 2).  Rows behind a sequence's last key are read from that key and masked.
//
// Batch invariance: a tile's keys, blocks and order follow from its own sequence's lengths, and the variant from
// sizes that a call's sequences share.
//
// What bounds it: the vector units and the matrix cores in turn.  A score costs about seven vector slots
// (maximum, fused multiply-add, exponential at a quarter of the rate, conversion, sum) and 4 D / 1024 matrix cycles of
// a 16-bit type; two or three wavefronts of a SIMD overlap the two in part.  bf16, 16/4 heads of 128, 2 x 8192 tokens
// under a window of 2048: 286 us, 842 TF/s of visible pairs; fp16, 8/2 heads of 64, 32 packed prompts of 19533 tokens, window 256: 30 us.  float32 products
// run at 1/16 of the 16-bit rate and bound it alone: 3 x 257 rows of 1281 keys, 16 heads of 72, window 500: 37 us.
#include <type_traits>

#include "gemm_core.h"
#include "rowops.h"
#include "scores.h"

namespace biops {

constexpr int kWindowFew = 64;      // rows up to which two wavefronts share them (window_launch_rows)
// Keys of a range and ranges of a few rows at most (window_splits); a range has at least 16 keys for each of the rows, so that
// their partial results stay a part of the keys' and values' bytes.
constexpr int kWindowRange = 512, kWindowRanges = 16;
constexpr float kWindowSlack = 8.f;  // by how many powers of two weights may pass one (weigh)
// A weight is 2^(c s - c m) by one fused multiply-add with c m rounded.  The rounding is the same factor in all weights of a
// row, and no more than 2^(1/16) up to this size of c m; past it the difference s - m is taken first (with an instruction
// more), or the factor would leave the range: by 2^28 fp16's, by 2^31 float's.
constexpr float kWindowLarge = 0x1p20f;
// fp16 weights are 2^7 times their size, which with the slack is near the end of their range: those down to 2^-32 of the largest
// count (2^-25 without it, which 100000 keys add up to 2^-8 of a row).
template <typename T> constexpr float kWindowUp = std::is_same<T, f16_t>::value ? 7.f : 0.f;
// Weights of mode 2 are 2^-40 times their size: of fewer than 2^31 values times weights of up to 2^kWindowSlack no sum passes
// the largest one.
constexpr float kWindowDown = 40.f;
template <typename T> constexpr int kWindowLast = std::is_same<T, f16_t>::value ? 1 : 2;  // (no sum of fp16 values passes float's range)
constexpr int kWindowOrder = 512;  // tiles that are dealt to the XCDs in runs

struct WindowArgs {
  const char *q, *k, *v;
  char* out;
  int64_t qB, qT, qH, kB, kT, kH, vB, vT, vH, oB, oT, oH;  // byte strides: batch, token, head
  const void *cu_q, *cu_k;  // packed: offsets [nseq + 1]; dense: null
  int cu_q64, cu_k64;
  int64_t cu_q_stride, cu_k_stride;
  int* flag;
  int64_t nseq;             // sequences (batch)
  uint32_t first, total;    // first tile of a launch; tiles of the call
  int lq, lk;               // dense lengths; packed: all query and key rows
  uint32_t tiles;           // dense: tiles of a sequence; packed: most tiles of a head
  uint32_t hkv, group;
  int d, dv;
  int splits, per;          // ranges of keys that a tile's workgroups take, blocks of a range
  float *part, *ml;         // their results: [row][range][dv], [row][range][2]
  int window, sinks;        // window >= 1 (2^31 - 1: all)
  int negate, zero;         // the scale is negative, or 0 (score_scale)
  float scale;              // c > 0
};

struct WindowTile {
  int qrow, krow;      // first row of the sequence in the packed tensors (0 in dense)
  int ql, kl;          // lengths
  int i0;              // first row of the tile in its sequence
};

__device__ __forceinline__ int64_t window_offset(const void* cu, int is64, int64_t stride, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(cu)[i * stride] : (int64_t) reinterpret_cast<const int32_t*>(cu)[i * stride];
}

template <typename T>
__device__ __forceinline__ uint32_t window_pack(float x, float y) {
  if constexpr (std::is_same<T, bf16_t>::value) return f32x2_to_bf16x2_bits(x, y);
  else return f32x2_to_f16x2_bits(x, y);
}
// l + x + y of a packed pair: the sum is of the rounded weights, which the product takes, at one instruction for two.
template <typename T>
__device__ __forceinline__ float window_add_pair(uint32_t xy, float l) {
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, xy), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, xy), __builtin_bit_cast(f16x2_t, 0x3c003c00u), l, false);
}

// Tile `tl` of the packed rows.  Segment 0 are rows in front of the first offset, segment j sequence j - 1, the last one
// the rows behind the last offset; the outer two have no keys and become zeros.  Segment j's tiles are numbered from
// begin / ROWS + j: that leaves room for as many as it can need, without counting those in front of it, so the
// segment is found by a search, 64 places at a time.  Offsets are taken into [0, rows]; where they do not rise the search
// ends somewhere, and what it finds is inside the tensors.
template <int ROWS>
__device__ __forceinline__ bool window_find(const WindowArgs& a, int tl, int lane, WindowTile& t) {
  const int n = (int)a.nseq;
  int at = 0, left = n + 2;  // segments that are left to choose from
  for (;;) {
    const int step = (left - 1) / 64 + 1;
    const bool in = lane < (left - 1) / step + 1;
    const int j = at + (in ? lane * step : 0);
    int64_t qs = 0, qe = a.lq, ks = 0, ke = -1;
    if (j >= 1) qs = window_offset(a.cu_q, a.cu_q64, a.cu_q_stride, j - 1);
    if (step == 1) {  // what the last round needs, fetched along
      if (j <= n) qe = window_offset(a.cu_q, a.cu_q64, a.cu_q_stride, j);
      if (j >= 1 && j <= n) {
        ks = window_offset(a.cu_k, a.cu_k64, a.cu_k_stride, j - 1);
        ke = window_offset(a.cu_k, a.cu_k64, a.cu_k_stride, j);
      }
    }
    auto row = [&](int64_t x) -> int { return x < 0 ? 0 : (x > a.lq ? a.lq : (int)x); };
    const int begin = row(qs), rows = row(qe) - begin;
    const int tile = tl - (begin / ROWS + j);
    const uint64_t hit = __ballot(in && tile >= 0);
    if (hit == 0) return false;
    const int f = 63 - __builtin_clzll(hit);
    if (step == 1) {
      const bool keys_ok = ks >= 0 && ke >= ks && ke <= a.lk;
      t.qrow = __builtin_amdgcn_readlane(begin, f);
      t.ql = __builtin_amdgcn_readlane(rows, f);
      t.krow = __builtin_amdgcn_readlane(keys_ok ? (int)ks : 0, f);
      t.kl = __builtin_amdgcn_readlane(keys_ok ? (int)(ke - ks) : 0, f);
      const int64_t i0 = (int64_t)__builtin_amdgcn_readlane(tile, f) * ROWS;
      t.i0 = (int)i0;
      return i0 < t.ql;
    }
    at += f * step;
    left = step < left - f * step ? step : left - f * step;
  }
}

// Whether sequence i's offsets rise and stay inside the tensors (i = nseq: whether the first ones are zero and the last one
// of the queries inside).
__device__ __forceinline__ bool window_offsets_ok(const WindowArgs& a, int64_t i) {
  auto q = [&](int64_t x) { return window_offset(a.cu_q, a.cu_q64, a.cu_q_stride, x); };
  auto k = [&](int64_t x) { return window_offset(a.cu_k, a.cu_k64, a.cu_k_stride, x); };
  if (i == a.nseq) return q(0) == 0 && k(0) == 0 && q(i) <= a.lq;
  const int64_t ks = k(i), ke = k(i + 1);
  return q(i) <= q(i + 1) && ks >= 0 && ks <= ke && ke <= a.lk;
}

// The check alone, for calls without query rows or heads.
__global__ __launch_bounds__(256) void window_offsets_kernel(WindowArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i <= a.nseq && !window_offsets_ok(a, i)) *a.flag = 1;
}

// DP, DVP: head and value size rounded up to whole fragments; RW row groups of 32 (of HG heads) by KW wavefronts that
// share a row group and take turns at the keys.
template <typename T, int DP, int DVP, int RW, int KW_, int NH_, int HG>
struct WindowShape {
  static constexpr int E = sizeof(T), VEC = 16 / E;
  static constexpr int KW = KW_, NH = NH_;             // NH: 32-key parts of a block that a wavefront takes
  static constexpr int ROWS = 32 * RW / HG, THREADS = 64 * RW * KW;
  static constexpr int BN = 32 * NH * KW;              // keys of a block
  static constexpr int KCH = DP / VEC, VCH = DVP / VEC;  // 16-byte chunks of a K / V row
  static constexpr int slots(int chunks) { return chunks <= 8 ? 8 : (chunks <= 16 ? 16 : 32); }
  static constexpr int KS = slots(KCH), VS = slots(VCH);  // ... and their places in LDS
  static constexpr int K_BYTES = BN * KS * 16, V_BYTES = BN * VS * 16;
  // A thread loads chunk slot tid % KS of every KRth row.
  static constexpr int KR = THREADS / KS, VR = THREADS / VS;
  static constexpr int KL = BN / KR, VL = BN / VR;
  static constexpr int QF = DP / (2 * VEC);            // fragment steps of a 32x32 score block
  static constexpr int QSTEP = 4 / NH;                 // score steps whose fragments are read at a time
  static constexpr int OF = (DVP + 31) / 32;
  static constexpr int JOIN_BYTES = KW > 1 ? (KW - 1) * RW * 64 * (16 * OF + 2) * 4 : 0;
  static constexpr int BLOCK_BYTES = K_BYTES + V_BYTES;
  static constexpr int LDS_BYTES = BLOCK_BYTES > JOIN_BYTES ? BLOCK_BYTES : JOIN_BYTES;
  static_assert(BN % KR == 0 && BN % VR == 0, "whole loads");
  static_assert(32 * OF <= VS * VEC, "V fragments stay inside a row");
  // Place of chunk c in row r: K so that sixteen consecutive rows of one chunk lie in sixteen different 16-byte
  // slots, V as the transposing reads want it (float32: rows r and r + 4 in opposite halves of the banks).
  __device__ static __forceinline__ int k_slot(int r, int c) { return KS >= 16 ? c ^ (r & 15) : c ^ ((r >> 1) & 7); }
  __device__ static __forceinline__ int v_slot(int r, int c) {
    return E == 2 ? c ^ nmajor_swz<VS>(r) : c ^ nmajor32_swz<VS>(r);
  }
  __device__ static __forceinline__ int k_off(int r, int c) { return (r * KS + k_slot(r, c)) << 4; }
  __device__ static __forceinline__ int v_off(int r, int col) {
    return ((r * VS + v_slot(r, col / VEC)) << 4) + (col % VEC) * E;
  }
};

// c m as weights take it off, less the powers of two that these are larger by; c = a.scale.
template <typename T>
__device__ __forceinline__ float window_shift(float m, float c) {
  if constexpr (kWindowUp<T> == 0.f) return m * c;
  else return __builtin_fmaf(m, c, -kWindowUp<T>);
}
// Exponent that turns weights relative to the score m into those relative to the score top.  (The shifts are the rounded ones
// that the weights have seen: no fused multiply-add may take their place.  `exact`: mode 2, where all differences are
// taken first.)
template <typename T>
__device__ __forceinline__ float window_ratio(float m, float top, float c, bool exact) {
#pragma clang fp contract(off)
  const float a = window_shift<T>(m, c), t = window_shift<T>(top, c);
  const bool la = exact || fabsf(a) > kWindowLarge, lt = exact || fabsf(t) > kWindowLarge;
  if (!la && !lt) return a - t;
  auto rounding = [&](float x, float shift) { return __builtin_fmaf(x, c, -shift) - kWindowUp<T>; };
  return (m - top) * c - (la ? 0.f : rounding(m, a)) + (lt ? 0.f : rounding(top, t));
}

// Infinities and NaN of 16 bytes as zeros.
template <typename T>
__device__ __forceinline__ u32x4_t finite_or_zero(u32x4_t v) {
  constexpr uint32_t inf = score_inf<T>();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Num<T>::kBytes == 4) v[i] = (v[i] & inf) == inf ? 0u : v[i];
    else v[i] = ((v[i] & inf) == inf ? 0u : v[i] & 0xffffu) | ((v[i] & inf << 16) == inf << 16 ? 0u : v[i] & 0xffff0000u);
  }
  return v;
}

// What a wavefront's part of a tile is (the same for all its lanes).
struct WindowPart {
  WindowTile tile;
  int64_t b;
  int h, w, range;  // head, wavefront of the workgroup, range of keys
};

// The keys of a tile, counted through from 0: v is key v < ns ? v : v + shift (sinks, then everything from the first row's
// window on).
struct WindowKeys {
  int p0, qrows;     // position of the tile's first row; its rows
  int ns, shift, nv; // nv: how many there are
  int sv;            // every row sees v < sv, up to its own position: sinks
  int blk0, nblk;    // blocks that the workgroup takes
};
__device__ __forceinline__ WindowKeys window_keys(const WindowArgs& a, const WindowPart& part, int rows, int block) {
  const WindowTile& tile = part.tile;
  WindowKeys k;
  k.qrows = tile.ql - tile.i0 < rows ? tile.ql - tile.i0 : rows;
  k.p0 = tile.kl - tile.ql + tile.i0;
  const int p1 = k.p0 + k.qrows - 1;
  const int64_t begin = (int64_t)k.p0 - a.window + 1;
  const int start = begin > 0 ? (int)begin : 0;
  k.ns = tile.kl > 0 ? (a.sinks < start ? a.sinks : start) : 0;
  k.shift = start - k.ns;
  k.nv = tile.kl > 0 && p1 >= 0 ? p1 + 1 - k.shift : 0;
  const int all = (k.nv + block - 1) / block;
  k.blk0 = part.range * a.per;
  k.nblk = a.per < all - k.blk0 ? k.blk0 + a.per : all;
  // (sinks in front of the first row's window are before every row; the others are among the window's keys)
  k.sv = k.shift > 0 ? k.ns : a.sinks;
  return k;
}

// Infinities and NaN among the values that rows see, set in their outputs whatever the weights: +inf and -inf in one column
// make NaN.  Rows `odd` of the wavefront's 32.  A lane keeps a bit for each of them in its columns.
template <typename T, int OF>
__device__ __forceinline__ void window_mark(const WindowArgs& a, const WindowPart& part, int r0, int rows, int block, uint32_t odd, int lane) {
  constexpr int N = (OF + 1) / 2, AHEAD = 8;
  const WindowKeys keys = window_keys(a, part, rows, block);
  const char* const v = a.v + part.b * a.vB + part.tile.krow * a.vT + part.h / (int)a.group * a.vH;
  const int first = keys.blk0 * block, last = keys.nblk * block < keys.nv ? keys.nblk * block : keys.nv;
  const int64_t hi = (int64_t)keys.p0 + r0 - keys.shift;  // the last counted key that row 0 sees
  uint32_t up[N], down[N];
#pragma unroll
  for (int i = 0; i < N; ++i) up[i] = down[i] = 0u;
  auto below = [](int64_t n) -> uint32_t { return n <= 0 ? 0u : ~0u >> (n < 32 ? 32 - n : 0); };  // the n lowest bits
#pragma unroll 1
  for (int k = first; k < last; k += AHEAD) {
    float x[AHEAD][N];
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {
      const int c = k + t < last ? k + t : last - 1;
      const T* row = reinterpret_cast<const T*>(v + (int64_t)(c < keys.ns ? c : c + keys.shift) * a.vT);
#pragma unroll
      for (int i = 0; i < N; ++i) x[t][i] = lane + 64 * i < a.dv ? Num<T>::load(row + lane + 64 * i) : 0.f;
    }
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {
      const int64_t c = k + t < last ? k + t : last - 1;
      const uint32_t see = odd & ~below(c - hi) & (c < keys.sv ? ~0u : below(c + a.window - hi));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!(x[t][i] < INFINITY)) up[i] |= see;  // (NaN: both)
        if (!(x[t][i] > -INFINITY)) down[i] |= see;
      }
    }
  }
  auto store = [&](auto* to, int64_t step) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int col = lane + 64 * i;
      if (col >= a.dv) continue;
      for (uint32_t rest = up[i] | down[i]; rest != 0; rest &= rest - 1) {
        const int r = __builtin_ctz(rest);
        const float x = (up[i] & down[i]) >> r & 1 ? NAN : (up[i] >> r & 1 ? INFINITY : -INFINITY);
        Num<std::remove_pointer_t<decltype(to)>>::store(to + r * step + col, x);
      }
    }
  };
  if (a.splits > 1) {
    const int64_t row = (part.b * (a.hkv * a.group) + part.h) * a.lq + part.tile.i0 + r0;
    store(a.part + (row * a.splits + part.range) * a.dv, (int64_t)a.splits * a.dv);
  } else {
    char* const out = a.out + part.b * a.oB + (int64_t)(part.tile.qrow + part.tile.i0 + r0) * a.oT + part.h * a.oH;
    store(reinterpret_cast<T*>(out), a.oT / (int64_t)sizeof(T));
  }
}

// Wavefronts per SIMD that registers are given out for.
template <typename T, int DP, int DVP, int NH>
constexpr int window_waves() {
  return DP > 128 || DVP > 128 ? 1 : (sizeof(T) == 2 && DP <= 64 && DVP <= 64 ? (NH == 1 ? 4 : 3) : 2);
}

// Rows `left` of the wavefront's 32 in one pass over the tile's keys, stored.  Returns those without a result, which take
// another mode.  Mode 0 is a function of its own (AGAIN false), so that what the others need costs it no registers.
template <typename T, int DP, int DVP, int RW, int KW, int NH, int HG, bool AGAIN>
__device__ __forceinline__ uint32_t window_pass(const WindowArgs& a, char* smem, const WindowPart& own_part, int tid, uint32_t left, int mode_) {
  using F = WindowShape<T, DP, DVP, RW, KW, NH, HG>;
  constexpr int E = F::E, BN = F::BN;
  const int mode = AGAIN ? mode_ : 0;
  const WindowTile& tile = own_part.tile;
  const int64_t b = own_part.b;
  const int w = own_part.w, h = own_part.h, hk = h / (int)a.group, range = own_part.range;
  const int lane = tid & 63, hf = lane >> 5, l32 = lane & 31;
  const int rw = w % RW, part = w / RW;  // row group, turn at the keys
  const int r0 = 32 * (rw / HG);         // its first row
  const u32x4_t zero4 = {0u, 0u, 0u, 0u};
  const WindowKeys keys = window_keys(a, own_part, F::ROWS, BN);
  const int qrows = keys.qrows, p0 = keys.p0, ns = keys.ns, shift = keys.shift, nv = keys.nv;
  const int blk0 = keys.blk0, nblk = keys.nblk;
  const char* const qb = a.q + b * a.qB + (int64_t)(tile.qrow + tile.i0) * a.qT + h * a.qH;
  const char* const kb = a.k + b * a.kB + tile.krow * a.kT + hk * a.kH;
  const char* const vb = a.v + b * a.vB + tile.krow * a.vT + hk * a.vH;
  char* const ob = a.out + b * a.oB + (int64_t)(tile.qrow + tile.i0) * a.oT + h * a.oH;

  // What a row sees of the counted keys: lo .. hi (its window), and v < sv (sinks; cut off at hi).
  const int sv = keys.sv;
  auto row_lo = [&](int p) -> int {
    const int64_t x = (int64_t)p - a.window + 1 - shift;
    return x > 0 ? (int)x : 0;
  };

  const int rloc = r0 + l32;
  const bool row_ok = rloc < qrows;
  const int hi = row_ok ? p0 + rloc - shift : -1;  // negative: nothing
  const int lo = row_lo(p0 + rloc);
  const int wlast = r0 + 31 < qrows ? r0 + 31 : qrows - 1;  // last row of the wavefront
  const bool wany = r0 < qrows;
  const int wlo0 = row_lo(p0 + r0), wlo1 = row_lo(p0 + wlast);
  const int whi0 = p0 + r0 - shift, whi1 = p0 + wlast - shift;

  // Rows behind the last one take its queries; they see nothing.
  u32x4_t qf[F::QF];
  {
    const char* qr = qb + (row_ok ? rloc : qrows - 1) * a.qT;
    if (a.d == DP) {
#pragma unroll
      for (int c = 0; c < F::QF; ++c) qf[c] = load_16(qr + 16 * (2 * c + hf));
    } else {
#pragma unroll
      for (int c = 0; c < F::QF; ++c) qf[c] = F::VEC * (2 * c + hf) < a.d ? load_16(qr + 16 * (2 * c + hf)) : zero4;
    }
    if (a.negate | a.zero) {
#pragma unroll
      for (int c = 0; c < F::QF; ++c) qf[c] = score_query<T>(qf[c], a.negate, a.zero);
    }
  }

  // Blocks go from memory straight to LDS (16 bytes a lane, at consecutive places: the lane that fills slot x of a
  // row fetches the chunk whose place that is).  Chunks behind the head size are zeroed once and stay.
  // (Rows of 32 slots: a thread's rows alternate between two K chunks.)
  constexpr int KV = F::KS >= 16 && F::KR < 16 ? 2 : 1;
  const int krow = tid / F::KS, vrow0 = tid / F::VS, vc = F::v_slot(vrow0, tid % F::VS);
  int kc[KV];
  bool kin[KV];
  uint32_t koff[KV];
#pragma unroll
  for (int j = 0; j < KV; ++j) {
    kc[j] = F::k_slot(krow + F::KR * j, tid % F::KS);
    kin[j] = F::VEC * kc[j] < a.d;
    koff[j] = (uint32_t)(krow * (int)a.kT + 16 * kc[j]);
  }
  const bool vin = F::VEC * vc < a.dv;
  const uint32_t voff = (uint32_t)(vrow0 * (int)a.vT + 16 * vc);
  char* const kbuf = smem;
  char* const vbuf = smem + F::K_BYTES;
  // Row v of the counted keys; behind the last one, that one (no row sees it there).
  auto key_of = [&](int v) -> int64_t {
    v = v < nv ? v : nv - 1;
    return v < ns ? v : v + shift;
  };
  auto fetch = [&](const char* from, char* to) {
    __builtin_amdgcn_global_load_lds((global_cvoid_t*)from, (lds_void_t*)to, 16, 0, 0);
  };
  auto load_k = [&](int blk) {
    const int v0 = blk * BN;
    char* to = kbuf + w * 1024;
    const bool whole = v0 >= ns && v0 + BN <= nv;
    const char* kp = kb + (int64_t)(v0 + shift) * a.kT;
#pragma unroll
    for (int j = 0; j < KV; ++j) {
      if (!kin[j]) continue;
      if (whole) {
#pragma unroll
        for (int i = j; i < F::KL; i += KV) fetch(kp + i * (F::KR * a.kT) + koff[j], to + 16 * F::THREADS * i);
      } else {
#pragma unroll
        for (int i = j; i < F::KL; i += KV) fetch(kb + key_of(v0 + krow + F::KR * i) * a.kT + 16 * kc[j], to + 16 * F::THREADS * i);
      }
    }
  };
  auto load_v = [&](int blk) {
    if (!vin) return;
    const int v0 = blk * BN;
    char* to = vbuf + w * 1024;
    if (v0 >= ns && v0 + BN <= nv) {
      const char* vp = vb + (int64_t)(v0 + shift) * a.vT;
#pragma unroll
      for (int i = 0; i < F::VL; ++i) fetch(vp + i * (F::VR * a.vT) + voff, to + 16 * F::THREADS * i);
    } else {
#pragma unroll
      for (int i = 0; i < F::VL; ++i) fetch(vb + key_of(v0 + vrow0 + F::VR * i) * a.vT + 16 * vc, to + 16 * F::THREADS * i);
    }
  };
  // Everything fetched and every LDS read has landed, in all wavefronts.
  auto meet = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (a.d < F::KS * F::VEC || a.dv < F::VS * F::VEC) {
#pragma unroll
    for (int i = 0; i < F::KL; ++i)
      if (!kin[i % KV]) *reinterpret_cast<u32x4_t*>(kbuf + 16 * tid + 16 * F::THREADS * i) = zero4;
    if (!vin) {
#pragma unroll
      for (int i = 0; i < F::VL; ++i) *reinterpret_cast<u32x4_t*>(vbuf + 16 * tid + 16 * F::THREADS * i) = zero4;
    }
  }

  // m: the score (raw) that weights are relative to, sh = window_shift of it (0 before the first), l: this lane's part of the row's sum
  float m = -INFINITY, sh = 0.f, l = 0.f;
  const float slack = fminf(kWindowSlack / a.scale, FLT_MAX);
  f32x16_t oacc[F::OF];  // O^T: register r of block e is column 32e + 8(r/4) + 4hf + r%4 of row l32
#pragma unroll
  for (int e = 0; e < F::OF; ++e)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[e][r] = 0.f;

  const int hb0 = NH * part;  // this wavefront's 32-key parts of a block: hb0 .. hb0 + NH - 1
  f32x16_t sc[NH];
  auto scores = [&]() {
    const char* ks = kbuf;
#pragma unroll
    for (int x = 0; x < NH; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[x][r] = 0.f;
    // The fragments of a group of steps are read before the MFMAs of the group before it (the barriers keep the
    // compiler from sinking each read next to its MFMA, where it would show its latency).
    u32x4_t kf[2][F::QSTEP][NH];
    auto read = [&](int c0, int to) {
#pragma unroll
      for (int c = 0; c < F::QSTEP; ++c)
#pragma unroll
        for (int x = 0; x < NH; ++x)
          if (c0 + c < F::QF)
            kf[to][c][x] = *reinterpret_cast<const u32x4_t*>(ks + F::k_off(32 * (hb0 + x) + l32, 2 * (c0 + c) + hf));
    };
    read(0, 0);
#pragma unroll
    for (int g = 0; g * F::QSTEP < F::QF; ++g) {
      if ((g + 1) * F::QSTEP < F::QF) read((g + 1) * F::QSTEP, (g + 1) & 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < F::QSTEP; ++c)
#pragma unroll
        for (int x = 0; x < NH; ++x)
          if (g * F::QSTEP + c < F::QF && (E == 2 || 2 * F::VEC * (g * F::QSTEP + c) < a.d)) Mfma<T>::step(sc[x], kf[g & 1][c][x], qf[g * F::QSTEP + c]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Masks the scores of a block, rescales what is summed where a row's maximum grows, and turns scores into weights.
  u32x4_t pw[E == 2 ? NH : 1][2];  // 16-bit weights, packed; float32 ones stay in sc
  auto weigh = [&](int blk) {
    const int v0 = blk * BN + 32 * hb0, v1 = v0 + 32 * NH - 1;
    if (!(wlast == r0 + 31 && v0 >= wlo1 && v1 <= whi0)) {  // not all rows see all keys
      // A row's keys of a part as bits, so that a score costs one bit's extension and one selection.
      auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : ~0u >> (n < 32 ? 32 - n : 0); };  // the n lowest bits
#pragma unroll
      for (int x = 0; x < NH; ++x) {
        const int v = v0 + 32 * x;
        // register r: key 8(r/4) + 4hf + r%4
        const uint32_t seen = ((below(hi + 1 - v) & ~below(lo - v)) | below((sv <= hi ? sv : hi + 1) - v)) >> (4 * hf);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t keep = (uint32_t)((int32_t)(seen << (31 - (8 * (r >> 2) + (r & 3)))) >> 31);
          sc[x][r] = __uint_as_float((__float_as_uint(sc[x][r]) & keep) | (0xff800000u & ~keep));
        }
      }
    }
    float mx = sc[0][0];
#pragma unroll
    for (int x = 0; x < NH; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[x][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // A row's maximum is followed when it has grown by more than 2^kWindowSlack in its weights: until then they are that
    // much larger than one at most, and nothing is rescaled
    // (2 to 5 % of the time; 16 % with 256-wide heads and few rows).  Each row by itself, so that no row's bits depend on another.
    const bool grown = mx - m > slack;
    if (__any(grown)) {
      const float mn = grown ? mx : m;
      const float to = mn == -INFINITY ? 0.f : window_shift<T>(mn, a.scale);
      if (__any(m > -INFINITY)) {  // (nothing is summed before a row's first keys)
        const float corr = grown && m > -INFINITY ? __builtin_amdgcn_exp2f(window_ratio<T>(m, mn, a.scale, mode == 2)) : 1.f;
        l *= corr;
#pragma unroll
        for (int e = 0; e < F::OF; ++e)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[e][r] *= corr;
      }
      m = mn;
      sh = to;
    }
    const bool large = mode == 2 || fabsf(sh) > kWindowLarge;
    if (__any(large)) {
      const float less = large && m > -INFINITY ? m : 0.f;
#pragma unroll
      for (int x = 0; x < NH; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[x][r] -= less;
    }
    // A block's 16-bit weights are added up by themselves: one by one, those below 2^-25 of the sum so far would not count in
    // it, as they do in the product's sums, 16 keys at a time.  (float32 products add two keys at a time.)
    float sum = 0.f;
    const float off = large ? (mode == 2 ? kWindowDown : -kWindowUp<T>) : sh;
#pragma unroll
    for (int x = 0; x < NH; ++x) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][r], a.scale, -off));
        if constexpr (E == 4) l += sc[x][r];
      }
      if constexpr (E == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pw[x][i >> 2][i & 3] = window_pack<T>(sc[x][2 * i], sc[x][2 * i + 1]);
          sum = window_add_pair<T>(pw[x][i >> 2][i & 3], sum);
        }
      }
    }
    l += sum;
  };
  // What the weights add to the output.
  auto gather = [&]() {
    const char* vs = vbuf;
    if constexpr (E == 4) {
      // the values of a group of four steps are read before the MFMAs of the group before it
      float xv[2][4][F::OF];
      auto read = [&](int g, int to) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < F::OF; ++e)
            xv[to][r][e] = *reinterpret_cast<const float*>(vs + F::v_off(32 * hb0 + 8 * g + 4 * hf + r, 32 * e + l32));
      };
      read(0, 0);
#pragma unroll
      for (int g = 0; g < 4 * NH; ++g) {
        if (g + 1 < 4 * NH) read(g + 1, (g + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < F::OF; ++e)
            oacc[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(xv[g & 1][r][e], sc[g >> 2][4 * (g & 3) + r], oacc[e], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // Transposing reads: lane s of a 16-lane group points at row k0 + s/4, column n0 + 4(s%4), and receives rows
      // k0 .. k0+3 of column n0 + s.  In assembly, since the compiler would wait for all fetches before each; the
      // fragments of a 16-key step are read before the MFMAs of the step before it.
      const int vrow = 4 * hf + ((lane & 15) >> 2), vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      u32x2_t vl[2][F::OF], vh[2][F::OF];
      auto read = [&](int step, int to) {
        const int row = 32 * hb0 + 16 * step + vrow;
#pragma unroll
        for (int e = 0; e < F::OF; ++e) {
          vl[to][e] = lds_read_tr16_asm(vs + F::v_off(row, 32 * e + vcol));
          vh[to][e] = lds_read_tr16_asm(vs + F::v_off(row + 8, 32 * e + vcol));
        }
      };
      read(0, 0);
#pragma unroll
      for (int step = 0; step < 2 * NH; ++step) {
        const int at = step & 1;
#pragma unroll
        for (int e = 0; e < F::OF; ++e) lds_wait_anchor(vl[at][e], vh[at][e]);
        if (step + 1 < 2 * NH) read(step + 1, at ^ 1);
#pragma unroll
        for (int e = 0; e < F::OF; ++e)
          Mfma<T>::step(oacc[e], u32x4_t{vl[at][e][0], vl[at][e][1], vh[at][e][0], vh[at][e][1]}, pw[step >> 1][step & 1]);
      }
    }
  };
  // Whether any row of the wavefront sees a key of its part of a block.
  auto sees = [&](int blk) {
    const int v0 = blk * BN + 32 * hb0, v1 = v0 + 32 * NH - 1;
    return wany && blk < nblk && v0 <= whi1 && (v1 >= wlo0 || v0 < sv);
  };

  // A turn: weights of a block (vector work), then its product and the next block's scores (matrix work, at a
  // higher priority: of two wavefronts of a SIMD one multiplies while the other takes exponentials).  The block's values
  // and the next one's keys are fetched while the wavefronts weigh, when nothing reads the LDS.  Two buffers, filled a turn
  // ahead, were 2 to 12 % slower: every read's address then depends on the block, and so costs an instruction.
  if (blk0 < nblk) load_k(blk0);
  meet();
  bool here = sees(blk0);
  if (here) scores();
  for (int blk = blk0; blk < nblk; ++blk) {
    meet();
    load_v(blk);
    if (blk + 1 < nblk) load_k(blk + 1);
    if (here) weigh(blk);
    const bool then = sees(blk + 1);
    meet();
    if constexpr (AGAIN) {
      u32x4_t* const p = reinterpret_cast<u32x4_t*>(vbuf) + tid;
#pragma unroll 1
      for (int i = 0; i < F::VL; ++i) p[F::THREADS * i] = finite_or_zero<T>(p[F::THREADS * i]);
      meet();
    }
    __builtin_amdgcn_s_setprio(1);
    if (here) gather();
    if (then) scores();
    __builtin_amdgcn_s_setprio(0);
    here = then;
  }
  meet();

  l += __shfl_xor(l, 32, 64);
  if constexpr (KW > 1) {  // join the wavefronts of a row group, in order
    float* const js = reinterpret_cast<float*>(smem);
    if (part > 0) {
      float* o = js + ((part - 1) * RW + rw) * 64 * (16 * F::OF + 2) + lane;
#pragma unroll
      for (int e = 0; e < F::OF; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[64 * (16 * e + r)] = oacc[e][r];
      o[64 * 16 * F::OF] = m;
      o[64 * (16 * F::OF + 1)] = l;
    }
    __syncthreads();
    if (part == 0) {
      float top = m;
#pragma unroll
      for (int x = 1; x < KW; ++x) top = fmaxf(top, js[((x - 1) * RW + rw) * 64 * (16 * F::OF + 2) + lane + 64 * 16 * F::OF]);
      auto factor = [&](float from) {
        return from == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(window_ratio<T>(from, top, a.scale, mode == 2));
      };
      const float own = factor(m);
      l *= own;
#pragma unroll
      for (int e = 0; e < F::OF; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[e][r] *= own;
#pragma unroll
      for (int x = 1; x < KW; ++x) {
        const float* o = js + ((x - 1) * RW + rw) * 64 * (16 * F::OF + 2) + lane;
        const float f = factor(o[64 * 16 * F::OF]);
        l = __builtin_fmaf(o[64 * (16 * F::OF + 1)], f, l);
#pragma unroll
        for (int e = 0; e < F::OF; ++e)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[e][r] = __builtin_fmaf(o[64 * (16 * e + r)], f, oacc[e][r]);
      }
      m = top;
    }
  }
  uint32_t again = 0;
  if (part == 0) {
    if (__any(l == 0.f)) {  // rows that see nothing, or only scores of -inf
#pragma unroll
      for (int e = 0; e < F::OF; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[e][r] = l == 0.f ? 0.f : oacc[e][r];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // An output that is not finite over a finite sum: o * 0 is NaN.
    float odd = 0.f;
#pragma unroll
    for (int e = 0; e < F::OF; ++e)
#pragma unroll
      for (int r = 0; r < 16; ++r) odd = __builtin_fmaf(oacc[e][r], 0.f, odd);
    const uint64_t bad = __ballot(row_ok && l > 0.f && l < INFINITY && odd != 0.f);
    again = mode < kWindowLast<T> ? ((uint32_t)bad | (uint32_t)(bad >> 32)) & left : 0u;
    if (row_ok && (left & ~again) >> l32 & 1) {
      if constexpr (KW > 1) {
        if (a.splits > 1) {  // this range's part of the row: its own mean, and what that counts for
          const int64_t at = ((b * (a.hkv * a.group) + h) * a.lq + tile.i0 + rloc) * a.splits + range;
#pragma unroll
          for (int e = 0; e < F::OF; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int col = 32 * e + 8 * j + 4 * hf;
              if (col < a.dv)
                *reinterpret_cast<f32x4_t*>(a.part + at * a.dv + col) =
                    f32x4_t{oacc[e][4 * j] * inv, oacc[e][4 * j + 1] * inv, oacc[e][4 * j + 2] * inv, oacc[e][4 * j + 3] * inv};
            }
          if (hf == 0) {
            if (mode == 2) {  // as the weights of the other modes
              const float c = m * a.scale;
              l *= __builtin_amdgcn_exp2f(kWindowDown + (fabsf(c) > kWindowLarge ? 0.f : __builtin_fmaf(m, a.scale, -c)));
            }
            a.ml[2 * at] = m;
            a.ml[2 * at + 1] = l;
          }
        }
      }
      if (KW == 1 || a.splits == 1) {
        char* orow = ob + rloc * a.oT;
        auto put = [&](int e, int j) {
          const int col = 32 * e + 8 * j + 4 * hf;
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = oacc[e][4 * j + i] * inv;
          if constexpr (E == 4) {
            *reinterpret_cast<u32x4_any_t*>(orow + E * col) =
                u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
          } else {
            *reinterpret_cast<u32x2_any_t*>(orow + E * col) = u32x2_t{window_pack<T>(x[0], x[1]), window_pack<T>(x[2], x[3])};
          }
        };
        if (a.dv == 32 * F::OF) {
#pragma unroll
          for (int e = 0; e < F::OF; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) put(e, j);
        } else {
#pragma unroll
          for (int e = 0; e < F::OF; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (32 * e + 8 * j + 4 * hf < a.dv) put(e, j);
        }
      }
    }
  }
  return again;
}

// The part of wavefront w in workgroup `at` of the call; false where there is none.
template <int ROWS, int RW, int KW, int HG>
__device__ __forceinline__ bool window_part(const WindowArgs& a, uint32_t at, int w, int lane, WindowPart& p) {
  // Workgroups are dealt to the 8 XCDs in turn: every XCD takes a run of each kWindowOrder tiles, so that the
  // heads of a group and neighbouring tiles, which read the same keys, share one L2.
  uint32_t t = at;
  {
    const uint32_t first = t / kWindowOrder * kWindowOrder;
    const uint32_t n = a.total - first < kWindowOrder ? a.total - first : kWindowOrder;
    const uint32_t j = t - first;
    if ((n & 7) == 0) t = first + (j & 7) * (n >> 3) + (j >> 3);
  }
  p.w = w;
  p.range = 0;
  if constexpr (KW > 1) {
    if (a.splits > 1) {
      p.range = (int)(t % (uint32_t)a.splits);
      t /= (uint32_t)a.splits;
    }
  }
  const uint32_t tl = t % a.tiles;
  t /= a.tiles;
  const uint32_t htiles = a.hkv * a.group / HG;
  p.h = (int)(t % htiles) * HG + w % RW % HG;
  p.b = t / htiles;
  if (a.cu_q) {
    const bool work = window_find<ROWS>(a, (int)tl, lane, p.tile);
    if (p.h < HG && tl <= a.nseq && w == RW * KW - 1 && !window_offsets_ok(a, tl)) *a.flag = 1;
    return work;
  }
  p.tile.i0 = (int)(a.tiles - 1 - tl) * ROWS;  // longest ranges first
  p.tile.qrow = p.tile.krow = 0;
  p.tile.ql = a.lq;
  p.tile.kl = a.lk;
  return true;
}

template <typename T, int DP, int DVP, int RW, int KW, int NH, int HG>
__global__ __launch_bounds__(64 * RW * KW)
__attribute__((amdgpu_waves_per_eu(window_waves<T, DP, DVP, NH>(), window_waves<T, DP, DVP, NH>())))
void window_attn_kernel(WindowArgs a) {
  using F = WindowShape<T, DP, DVP, RW, KW, NH, HG>;
  __shared__ __attribute__((aligned(16))) char smem[F::LDS_BYTES];
  __shared__ int again_in[2];  // whether a row is left after mode 0, 1
  uint32_t odd;                // rows that were not finite in mode 0
  {
    const int tid = threadIdx.x;
    WindowPart p;  // (the wavefront's number is the same for its lanes, as the compiler is told)
    if (!window_part<F::ROWS, RW, KW, HG>(a, a.first + blockIdx.x, __builtin_amdgcn_readfirstlane(tid >> 6), tid & 63, p)) return;
    if (tid < 2) again_in[tid] = 0;
    odd = window_pass<T, DP, DVP, RW, KW, NH, HG, false>(a, smem, p, tid, ~0u, 0);
    if (odd != 0 && (tid & 63) == 0) again_in[0] = 1;
    __syncthreads();
    if (again_in[0] == 0) return;
  }
  // Arguments, thread and part are found again, so that none of them is kept in registers through the first pass.
  auto* at = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
  uint32_t block = blockIdx.x;
  int tid = threadIdx.x;
  asm volatile("" : "+s"(at), "+s"(block));
  asm volatile("" : "+v"(tid));
  uint32_t words[sizeof(WindowArgs) / 4];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(WindowArgs) / 4); ++i) words[i] = at[i];
  const WindowArgs again = __builtin_bit_cast(WindowArgs, words);
  WindowPart p;
  window_part<F::ROWS, RW, KW, HG>(again, again.first + block, __builtin_amdgcn_readfirstlane(tid >> 6), tid & 63, p);
  uint32_t left = odd;
#pragma unroll 1
  for (int mode = 1; mode <= kWindowLast<T>; ++mode) {
    left = window_pass<T, DP, DVP, RW, KW, NH, HG, true>(again, smem, p, tid, left, mode);
    if (mode == kWindowLast<T>) break;
    if (left != 0 && (tid & 63) == 0) again_in[mode] = 1;
    __syncthreads();
    if (again_in[mode] == 0) break;
  }
  if (odd != 0) {
    __builtin_amdgcn_s_waitcnt(0);  // the rows' stores come first
    window_mark<T, F::OF>(again, p, 32 * (p.w % RW / HG), F::ROWS, F::BN, odd, tid & 63);
  }
}

// Joins the ranges of one row per wavefront, in their order.
template <typename T>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t row = 4 * (a.first + blockIdx.x) + (threadIdx.x >> 6);
  if (row >= a.total) return;
  const int r = (int)(row % (uint32_t)a.lq);
  const uint32_t heads = a.hkv * a.group, h = row / (uint32_t)a.lq % heads;
  const int64_t b = row / (uint32_t)a.lq / heads;
  const float* const ml = a.ml + 2 * (int64_t)row * a.splits;
  const float* const part = a.part + (int64_t)row * a.splits * a.dv + 4 * lane;
  const float m = lane < a.splits ? ml[2 * lane] : -INFINITY, sum = lane < a.splits ? ml[2 * lane + 1] : 0.f;
  f32x4_t mean[kWindowRanges];  // on their way while the shares are found
#pragma unroll
  for (int x = 0; x < kWindowRanges; ++x)
    if (x < a.splits && 4 * lane < a.dv) mean[x] = *reinterpret_cast<const f32x4_t*>(part + (int64_t)x * a.dv);
  const float top = wave_max(m);
  // what each range's mean counts for
  const float own = m == -INFINITY ? 0.f : sum * __builtin_amdgcn_exp2f(window_ratio<T>(m, top, a.scale, false));
  const float l = wave_sum(own);
  const float share = l == 0.f ? 0.f : own / l;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < kWindowRanges; ++x)
    if (x < a.splits) o += mean[x] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(share), x));
  if (4 * lane >= a.dv) return;
  char* const out = a.out + b * a.oB + r * a.oT + h * a.oH;
#pragma unroll
  for (int i = 0; i < 4; ++i) Num<T>::store(reinterpret_cast<T*>(out) + 4 * lane + i, o[i]);
}

template <typename T, int DP, int DVP, int RW, int KW, int NH, int HG>
static int window_launch(WindowArgs a, hipStream_t s) {
  constexpr int rows = 32 * RW / HG;
  // packed: every sequence and the two ends may end in a part of a tile
  const int64_t tiles = a.cu_q ? a.lq / rows + a.nseq + 2 : cdiv(a.lq, rows);
  const int64_t heads = (int64_t)a.hkv * a.group / HG * (a.cu_q ? 1 : a.nseq);
  static_assert(KW == 1 || 32 * NH * KW == 64, "ranges are counted in blocks of 64 keys");
  if (tiles > INT64_C(0x7fffffff) / heads / a.splits) return fail(BIOPS_ERR_ARG, "biops_window_attention: more than 2^31 tiles");
  a.tiles = (uint32_t)tiles;
  a.total = (uint32_t)(tiles * heads * a.splits);
  constexpr uint32_t most = 1 << 22;  // a launch has less than 2^32 threads
  for (a.first = 0; a.first < a.total; a.first += most) {
    const uint32_t n = a.total - a.first < most ? a.total - a.first : most;
    hipLaunchKernelGGL((window_attn_kernel<T, DP, DVP, RW, KW, NH, HG>), dim3(n), dim3(64 * RW * KW), 0, s, a);
    const int rc = check_launch("window_attn_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  if (a.splits == 1) return BIOPS_OK;
  a.total = (uint32_t)(a.nseq * a.hkv * a.group * a.lq);
  const uint32_t groups = (a.total + 3) / 4;
  for (a.first = 0; a.first < groups; a.first += most) {
    const uint32_t n = groups - a.first < most ? groups - a.first : most;
    hipLaunchKernelGGL((window_join_kernel<T>), dim3(n), dim3(256), 0, s, a);
    const int rc = check_launch("window_join_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}
// What a workgroup takes.  Only sizes that all sequences of a call share may enter: the rows of a tile decide where
// its blocks of keys begin, and so the bits.
//
// Heads of a group in one workgroup share its fetches, and their tile of fewer rows has fewer keys that only some of its
// rows see.  Two wavefronts for the same rows, with the keys in turns, halve a tile's time where there are too few
// tiles to fill the chip, and cost their join; with float32 they win throughout.  us, variants as <wavefronts for rows and
// heads, turns, 32-key parts, heads>, 16/4 heads and a window of 512 unless said otherwise:
//   16-bit                           <4,1,2,4> <4,1,2,2> <4,1,2,1> <2,2,1,2> <2,2,1,1>
//   64-wide, 4 x 2048                  37.1      42.3      46.7      38.4      41.2
//   128-wide / 256-wide, the same     52 / 154  56 / 166  61 / 184  71 / 217  77 / 234
//   64-wide, 8/4 heads, all keys                 46.4      46.9      43.9      54.2
//   128-wide, 8/4 heads, w. 512 / all           30 / 66   33 / 66   39 / 61   42 / 79
//   64-wide, 8/8 heads, w. 64 / all                       13 / 47             13 / 54
//   128-wide, 8/8 heads, w. 512 / all                     34 / 66             42 / 79
//   64-wide, 50 rows of 700 keys, 1 / 64 sequences
//                                     16 / 23   16 / 23   15 / 33   12 / 25   12 / 24
//   128-wide, the same                20 / 33   20 / 32   19 / 45   16 / 41   16 / 41
//   float32 (<4,1,1,1>, without turns, beside them)          <4,1,1,1> <2,2,1,2> <2,2,1,1>
//   64-wide, 1 x 700 / 4 x 2048                              55 / 191  28 / 165  30 / 187
//   72-wide, the same                                        69 / 251  37 / 224  40 / 256
template <typename T, int DP>
static int window_launch_rows(const WindowArgs& a, hipStream_t s) {
  const bool pairs = a.group % 2 == 0, fours = a.group % 4 == 0;
  const bool few = !a.cu_q && a.lq <= kWindowFew;
  if (pairs && (sizeof(T) == 4 || few || (DP <= 64 && !fours))) return window_launch<T, DP, DP, 2, 2, 1, 2>(a, s);
  if (sizeof(T) == 4 || few) return window_launch<T, DP, DP, 2, 2, 1, 1>(a, s);
  if constexpr (sizeof(T) == 2) {
    if (fours) return window_launch<T, DP, DP, 4, 1, 2, 4>(a, s);
    if constexpr (DP > 64) {
      if (pairs) return window_launch<T, DP, DP, 4, 1, 2, 2>(a, s);
    }
    return window_launch<T, DP, DP, 4, 1, 2, 1>(a, s);
  } else {
    return BIOPS_OK;  // not reached
  }
}
template <typename T>
static int window_launch_d(const WindowArgs& a, hipStream_t s) {
  const int d = a.d > a.dv ? a.d : a.dv;
  if constexpr (sizeof(T) == 2) {
    if (d > 128) return window_launch_rows<T, 256>(a, s);
  }
  if (d <= 64) return window_launch_rows<T, 64>(a, s);
  if constexpr (sizeof(T) == 4) {
    if (d <= 80) return window_launch_rows<T, 80>(a, s);
  }
  if (d <= 96) return window_launch_rows<T, 96>(a, s);
  return window_launch_rows<T, 128>(a, s);
}

// Ranges that the keys of a few dense rows are cut into, by sizes that all sequences of a call share; blocks of 64 keys
// of a range.  A few rows are a few tiles, and each would walk through all keys alone.  us (one tile through all keys /
// ranges), bf16, 16/4 heads of 128, no window: 16 rows before 2000 keys 39 / 21 (one sequence), 40 / 23 (eight), 61 / 83
// (64); before 8192 keys 143 / 19, 144 / 42, 254 / 327; 64 rows before 8192 keys 133 / 26, 136 / 65, 445 / 538; float32,
// 72-wide, 16 rows before 8192 443 / 37, 443 / 114, 806 / 882.  (The batch may not enter: one sequence's bits.)
static int window_splits(int64_t lq, int64_t lk, int64_t window, int64_t sinks, int* per) {
  *per = 0x7fffffff;
  if (lq < 1 || lq > kWindowFew) return 1;
  const int64_t n = window < lk && sinks < lk - window ? (window + sinks + lq < lk ? window + sinks + lq : lk) : lk;
  const int64_t each = 16 * lq > kWindowRange ? 16 * lq : kWindowRange;
  if (n < 2 * each) return 1;
  const int64_t blocks = (n + 63) / 64, most = n / each < kWindowRanges ? n / each : kWindowRanges;
  *per = (int)((blocks + most - 1) / most);
  return (int)((blocks + *per - 1) / *per);
}

}  // namespace biops

using namespace biops;

extern "C" int64_t biops_window_attention_workspace_size(int64_t nseq, int64_t hq, int64_t lq, int64_t lk, int64_t dv,
                                                         int64_t window, int64_t sinks) {
  if (nseq < 0 || hq < 0 || lq < 0 || lk < 0 || dv < 0 || dv > 256 || window < 1 || sinks < 0 || hq > 65536 ||
      lk > INT64_C(0x7fffffff))
    return -1;
  int per;
  const int splits = window_splits(lq, lk, window, sinks, &per);
  if (splits == 1 || nseq == 0 || hq == 0) return 0;
  if (nseq > (INT64_C(1) << 30) / (hq * lq)) return -1;
  return nseq * hq * lq * splits * (dv + 2) * (int64_t)sizeof(float);
}

extern "C" int biops_window_attention_max_head(int dtype) {
  return dtype == BIOPS_F32 ? 128 : (dtype == BIOPS_F16 || dtype == BIOPS_BF16 ? 256 : 0);
}

extern "C" int biops_window_attention(int dtype, int64_t nseq, int64_t hq, int64_t hkv, int64_t lq, int64_t lk, int64_t d,
                                      int64_t dv, const void* q, int64_t sqB, int64_t sqT, int64_t sqH, const void* k,
                                      int64_t skB, int64_t skT, int64_t skH, const void* v, int64_t svB, int64_t svT,
                                      int64_t svH, void* out, int64_t soB, int64_t soT, int64_t soH, const void* cu_q,
                                      int cu_q64, int64_t cu_q_stride, const void* cu_k, int cu_k64, int64_t cu_k_stride,
                                      int64_t window, int64_t sinks, float scale, int* flag, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int elt = is_float_dtype(dtype) ? dtype_bytes(dtype) : 0;
  if (elt == 0) return fail(BIOPS_ERR_DTYPE, "biops_window_attention: unsupported dtype %d", dtype);
  if (nseq < 0 || hq < 0 || hkv <= 0 || hq % hkv != 0 || hq > 65536 || lq < 0 || lk < 0)
    return fail(BIOPS_ERR_ARG, "biops_window_attention: bad batch, heads or lengths");
  const int vec = 16 / elt, most = biops_window_attention_max_head(dtype);
  if (d < vec || d > most || d % vec || dv < vec || dv > most || dv % vec)
    return fail(BIOPS_ERR_ARG, "biops_window_attention: head sizes are multiples of %d up to %d", vec, most);
  if (window < 1 || sinks < 0) return fail(BIOPS_ERR_ARG, "biops_window_attention: window must be positive, sinks not negative");
  if (!(scale - scale == 0.f)) return fail(BIOPS_ERR_ARG, "biops_window_attention: scale is not finite");
  const int64_t longest = INT64_C(0x7fffffff) - 1024;  // tiles and blocks may round positions up
  if (lq > longest || lk > longest || nseq > longest) return fail(BIOPS_ERR_ARG, "biops_window_attention: more than 2^31 rows");
  // strides of a single element are never used
  if (cu_q || nseq == 1) skB = svB = 0;
  if (lk == 1) skT = svT = 0;
  if (hkv == 1) skH = svH = 0;
  // a block's rows are addressed by 32-bit offsets
  if (skT < 0 || svT < 0 || skT > (1 << 23) || svT > (1 << 23))
    return fail(BIOPS_ERR_LAYOUT, "biops_window_attention: key and value rows more than 2^23 elements apart");
  // ... and goes straight to LDS in 16-byte pieces
  if (lk > 0) {
    const int64_t all_k = (int64_t)reinterpret_cast<uintptr_t>(k) | elt * skB | elt * skT | elt * skH;
    const int64_t all_v = (int64_t)reinterpret_cast<uintptr_t>(v) | elt * svB | elt * svT | elt * svH;
    if ((all_k | all_v) & 15) return fail(BIOPS_ERR_LAYOUT, "biops_window_attention: keys or values not aligned to 16 bytes");
  }
  const bool empty = hq == 0 || lq == 0;
  if (!cu_q && (empty || nseq == 0)) return BIOPS_OK;
  if ((!empty && (!q || !out || (lk > 0 && (!k || !v)))) || (cu_q && (!cu_k || !flag)))
    return fail(BIOPS_ERR_ARG, "biops_window_attention: null pointer");
  WindowArgs a;
  a.q = static_cast<const char*>(q), a.k = static_cast<const char*>(k), a.v = static_cast<const char*>(v);
  a.out = static_cast<char*>(out);
  a.qB = elt * sqB, a.qT = elt * sqT, a.qH = elt * sqH;
  a.kB = elt * skB, a.kT = elt * skT, a.kH = elt * skH;
  a.vB = elt * svB, a.vT = elt * svT, a.vH = elt * svH;
  a.oB = elt * soB, a.oT = elt * soT, a.oH = elt * soH;
  a.cu_q = cu_q, a.cu_k = cu_k, a.cu_q64 = cu_q64 != 0, a.cu_k64 = cu_k64 != 0;
  a.cu_q_stride = cu_q_stride, a.cu_k_stride = cu_k_stride;
  a.flag = flag;
  a.nseq = nseq;
  a.lq = (int)lq, a.lk = (int)lk;
  if (empty) {
    hipLaunchKernelGGL(window_offsets_kernel, dim3((unsigned)(nseq / 256 + 1)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return check_launch("window_offsets_kernel");
  }
  a.hkv = (uint32_t)hkv, a.group = (uint32_t)(hq / hkv);
  a.d = (int)d, a.dv = (int)dv;
  const int64_t all = INT64_C(0x7fffffff);
  a.window = (int)(window < all ? window : all), a.sinks = (int)(sinks < all ? sinks : all);
  a.splits = 1, a.per = 0x7fffffff;
  a.part = a.ml = nullptr;
  if (!cu_q && lk > 0) {
    a.splits = window_splits(lq, lk, window, sinks, &a.per);
    if (a.splits > 1) {
      const int64_t need = biops_window_attention_workspace_size(nseq, hq, lq, lk, dv, window, sinks);
      if (need < 0) return fail(BIOPS_ERR_ARG, "biops_window_attention: more than 2^30 rows");
      if (!workspace || workspace_bytes < need)
        return fail(BIOPS_ERR_SIZE, "biops_window_attention: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
      if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BIOPS_ERR_LAYOUT, "biops_window_attention: workspace not 16-byte aligned");
      a.part = static_cast<float*>(workspace);
      a.ml = a.part + nseq * hq * lq * a.splits * dv;
    }
  }
  a.scale = score_scale(scale, &a.negate, &a.zero);
  BIOPS_DISPATCH_FLOAT(dtype, return window_launch_d<T>(a, static_cast<hipStream_t>(stream)));
  return BIOPS_OK;
}

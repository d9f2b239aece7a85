// Attention under a sliding window with a few first tokens (sinks) that stay visible: prompts and chunks
// of new tokens, dense [batch, heads, tokens, dim] or packed by sequence.
//
// Query r of a sequence (lq queries, lk keys) is the token at p = lk - lq + r and sees the keys j <= p
// with p - j < window or j < sinks:  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q.k_j.
//
// One workgroup (four wavefronts of 32 rows) owns 128 query rows of one head and passes once over the
// keys that any of them sees, counted through from 0: the sinks in front of the first row's window, then
// everything up to the last row.  So the sinks share the first block with the window's first keys, and work
// grows with the window, not with the sequence.  Blocks of 64 keys (32 in float32) go through LDS, double
// buffered; running maximum m and sum l per row, O rescaled when a maximum grows.
//
// Register layout: S^T = K Q^T (K as the A operand of 32x32 MFMAs) leaves lane L with query row L % 32 and
// keys 8j + 4(L/32) + i of a 32-key block, which is the B operand of O^T = V^T P^T with the same key order
// in V; so weights go from accumulators to the next MFMA without LDS, and a row's maximum, sum and rescale
// stay in its lane (one exchange between the two lanes of a row).  16-bit V fragments come from LDS by
// the transposing read.  16-bit weights are rounded once to the type for the product (half a step, as the
// output's own rounding); statistics and sums are 32-bit.
//
// A masked key never reaches a row.  Scores are replaced, not added to; keys past the sequence's end are
// zeros in LDS.  What is left is a value that is not finite at a key which one row of a block sees and
// another does not (0 * inf): a row whose sum is finite and whose output is not is computed again, key by
// key over what it sees (window_row).
//
// Batch invariance: a tile's keys, blocks and order follow from its own sequence's lengths alone.
#include <type_traits>

#include "gemm_core.h"
#include "rowops.h"

namespace biops {

constexpr int kWindowRows = 128;   // query rows of a workgroup
constexpr int kWindowOrder = 512;  // tiles that are dealt to the XCDs in runs

struct WindowArgs {
  const char *q, *k, *v;
  char* out;
  int64_t qB, qT, qH, kB, kT, kH, vB, vT, vH, oB, oT, oH;  // byte strides: batch, token, head
  const void *cu_q, *cu_k;  // packed: offsets [nseq + 1]; dense: null
  int cu_q64, cu_k64;
  int64_t cu_q_stride, cu_k_stride;
  int* flag;
  int64_t nseq, total;      // sequences (batch); workgroups' tiles
  int lq, lk;               // dense lengths; packed: all query and key rows
  int tiles;                // dense: tiles of a sequence; packed: most tiles of a head
  int hkv, group, d, dv;
  int window, sinks;        // window >= 1 (2^31 - 1: all)
  int negate;               // the scale is negative: queries enter with their sign flipped
  float scale;              // |scale| log2 e, > 0
};

struct WindowTile {
  int64_t qrow, krow;  // first row of the sequence in the packed tensors (0 in dense)
  int ql, kl;          // lengths
  int i0;              // first row of the tile in its sequence
};

__device__ __forceinline__ int64_t window_offset(const void* cu, int is64, int64_t stride, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(cu)[i * stride] : (int64_t) reinterpret_cast<const int32_t*>(cu)[i * stride];
}

// Tile `tl` of the packed rows.  Segment 0 are rows in front of the first offset, segment i sequence i - 1,
// the last one the rows behind the last offset; the outer two have no keys and become zeros.  Offsets are
// taken into [0, rows] and as their running maximum, so every row is in one segment whatever they hold.
__device__ __forceinline__ bool window_find(const WindowArgs& a, int tl, int lane, WindowTile& t) {
  const int n = (int)a.nseq, segments = n + 2;
  int before = 0, done = 0;  // end of the last segment, tiles so far
  for (int base = 0; base < segments; base += 64) {
    const int i = base + lane;
    const int64_t raw = i <= n ? window_offset(a.cu_q, a.cu_q64, a.cu_q_stride, i) : (int64_t)a.lq;
    int end = raw < 0 ? 0 : (raw > a.lq ? a.lq : (int)raw);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(end, o, 64);
      if (lane >= o && x > end) end = x;
    }
    if (before > end) end = before;
    if ((end != raw || (i == 0 && raw != 0))) *a.flag = 1;
    int begin = __shfl_up(end, 1, 64);
    if (lane == 0) begin = before;
    const int mine = (end - begin + kWindowRows - 1) / kWindowRows;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    upto += done;
    const uint64_t hit = __ballot(i < segments && upto > tl);
    if (hit != 0) {
      const int f = __builtin_ctzll(hit);
      const int b = __shfl(begin, f, 64), e = __shfl(end, f, 64), u = __shfl(upto, f, 64), m = __shfl(mine, f, 64);
      t.qrow = b;
      t.ql = e - b;
      t.i0 = (tl - (u - m)) * kWindowRows;
      t.krow = 0;
      t.kl = 0;
      const int seq = base + f - 1;
      if (seq >= 0 && seq < n) {
        const int64_t ks = window_offset(a.cu_k, a.cu_k64, a.cu_k_stride, seq), ke = window_offset(a.cu_k, a.cu_k64, a.cu_k_stride, seq + 1);
        if (ks >= 0 && ke >= ks && ke <= a.lk) {
          t.krow = ks;
          t.kl = (int)(ke - ks);
        } else {
          *a.flag = 1;
        }
      }
      return true;
    }
    before = __shfl(end, 63, 64);
    done = __shfl(upto, 63, 64);
  }
  return false;
}

template <typename T, int DP, int DVP>
struct WindowShape {
  static constexpr int E = sizeof(T), VEC = 16 / E;
  static constexpr int BN = E == 2 ? 64 : 32;          // keys of a block
  static constexpr int KCH = DP / VEC, VCH = DVP / VEC;  // 16-byte chunks of a K / V row
  static constexpr int K_BYTES = BN * DP * E, V_BYTES = BN * DVP * E;
  static constexpr int KL = BN * KCH / 256, VL = BN * VCH / 256;  // loads per thread and block
  static constexpr int QF = DP / (2 * VEC);            // fragment steps of a 32x32 score block
  static constexpr int OF = DVP / 32;
  static constexpr int NH = BN / 32;
  static_assert(BN * KCH % 256 == 0 && BN * VCH % 256 == 0, "whole loads");
  // chunk c of K row r: sixteen consecutive rows of one chunk in sixteen different 16-byte slots
  __device__ static __forceinline__ int k_off(int r, int c) {
    if constexpr (KCH >= 16) return r * (DP * E) + ((c ^ (r & 15)) << 4);
    else return r * (DP * E) + ((c ^ ((r >> 1) & 7)) << 4);
  }
  __device__ static __forceinline__ int v_off(int r, int col) {
    if constexpr (E == 2) return lds_off_n<VCH>(r, col);
    else return lds_off_n32<VCH>(r, col);
  }
};

// One row over exactly the keys that it sees, a wavefront together: the mean so far is kept normalised,
// so that values near the end of the type's range do not overflow either.
template <typename T>
__device__ __forceinline__ void window_row(const WindowArgs& a, const char* q, const char* k, const char* v, char* out,
                                           int p, int kl, int lane) {
  constexpr int MOST = 4;  // 256 / 64
  float x[MOST], o[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    x[i] = lane + 64 * i < a.d ? Num<T>::load(reinterpret_cast<const T*>(q) + lane + 64 * i) : 0.f;
    if (a.negate) x[i] = -x[i];
    o[i] = 0.f;
  }
  float sh = -INFINITY, l = 0.f;
  const int64_t start = (int64_t)p - a.window + 1;
  const int last = p < kl - 1 ? p : kl - 1;
  for (int j = 0; j <= last; ++j) {
    if (j >= a.sinks && j < start) {
      j = (int)start - 1;
      continue;
    }
    float s = 0.f;
    const T* kr = reinterpret_cast<const T*>(k + j * a.kT);
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (lane + 64 * i < a.d) s = __builtin_fmaf(x[i], Num<T>::load(kr + lane + 64 * i), s);
    s = wave_sum(s) * a.scale;
    if (s == -INFINITY) continue;
    const float top = fmaxf(sh, s);
    const float old = l * __builtin_amdgcn_exp2f(sh - top), add = __builtin_amdgcn_exp2f(s - top);
    l = old + add;
    sh = top;
    const float f = old / l, g = add / l;
    const T* vr = reinterpret_cast<const T*>(v + j * a.vT);
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (lane + 64 * i < a.dv) o[i] = __builtin_fmaf(Num<T>::load(vr + lane + 64 * i), g, o[i] * f);
  }
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (lane + 64 * i < a.dv) Num<T>::store(reinterpret_cast<T*>(out) + lane + 64 * i, o[i]);
}

template <int DP, int DVP>
constexpr int window_waves() { return DP > 128 || DVP > 128 ? 1 : 2; }

template <typename T, int DP, int DVP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(window_waves<DP, DVP>(), window_waves<DP, DVP>())))
void window_attn_kernel(WindowArgs a) {
  using F = WindowShape<T, DP, DVP>;
  constexpr int E = F::E, BN = F::BN, NH = F::NH;
  __shared__ __attribute__((aligned(16))) char smem[2 * (F::K_BYTES + F::V_BYTES)];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, hf = lane >> 5, l32 = lane & 31;
  const u32x4_t zero4 = {0u, 0u, 0u, 0u};

  for (int64_t turn = blockIdx.x; turn < a.total; turn += gridDim.x) {
    // Workgroups are dealt to the 8 XCDs in turn: every XCD takes a run of each kWindowOrder tiles, so that
    // the heads of a group and neighbouring tiles, which read the same keys, share one L2.
    int64_t t = turn;
    {
      const int64_t first = t / kWindowOrder * kWindowOrder;
      const int64_t n = a.total - first < kWindowOrder ? a.total - first : kWindowOrder;
      const int64_t j = t - first;
      if ((n & 7) == 0) t = first + (j & 7) * (n >> 3) + (j >> 3);
    }
    const int g = (int)(t % a.group);
    t /= a.group;
    WindowTile tile;
    int64_t b = 0;
    int hk;
    if (a.cu_q) {
      hk = (int)(t % a.hkv);
      if (!window_find(a, (int)(t / a.hkv), lane, tile)) continue;
    } else {
      tile.i0 = (a.tiles - 1 - (int)(t % a.tiles)) * kWindowRows;  // longest ranges first
      t /= a.tiles;
      hk = (int)(t % a.hkv);
      b = t / a.hkv;
      tile.qrow = tile.krow = 0;
      tile.ql = a.lq;
      tile.kl = a.lk;
    }
    const int h = hk * a.group + g;
    const int kl = tile.kl, qrows = tile.ql - tile.i0 < kWindowRows ? tile.ql - tile.i0 : kWindowRows;
    const char* const qb = a.q + b * a.qB + (tile.qrow + tile.i0) * a.qT + h * a.qH;
    const char* const kb = a.k + b * a.kB + tile.krow * a.kT + hk * a.kH;
    const char* const vb = a.v + b * a.vB + tile.krow * a.vT + hk * a.vH;
    char* const ob = a.out + b * a.oB + (tile.qrow + tile.i0) * a.oT + h * a.oH;

    // positions of the tile's first and last row; keys of v: v < ns ? v : v + shift
    const int p0 = kl - tile.ql + tile.i0, p1 = p0 + qrows - 1;
    const int64_t begin = (int64_t)p0 - a.window + 1;
    const int start = begin > 0 ? (int)begin : 0;
    const int ns = kl > 0 ? (a.sinks < start ? a.sinks : start) : 0;
    const int shift = start - ns;
    const int nv = kl > 0 && p1 >= 0 ? p1 + 1 - shift : 0;
    const int nblk = (nv + BN - 1) / BN;

    const int rloc = 32 * w + l32;
    const bool row_ok = rloc < qrows;
    const int p = p0 + rloc;                 // this lane's row
    const int wp0 = p0 + 32 * w;             // first and last position of the wavefront's rows
    const int wp1 = wp0 + 31 < p1 ? wp0 + 31 : p1;

    u32x4_t qf[F::QF];
#pragma unroll
    for (int c = 0; c < F::QF; ++c) {
      const int d0 = F::VEC * (2 * c + hf);
      qf[c] = row_ok && d0 < a.d ? load_16(qb + rloc * a.qT + E * d0) : zero4;
      if (a.negate) qf[c] ^= E == 2 ? 0x80008000u : 0x80000000u;
    }

    u32x4_t kr[F::KL], vr[F::VL];
    auto load = [&](int blk) {
      const int v0 = blk * BN;
      const bool whole = v0 >= ns && v0 + BN <= nv && a.d == DP && a.dv == DVP;
      if (whole) {
        const char* kp = kb + (int64_t)(v0 + shift) * a.kT;
        const char* vp = vb + (int64_t)(v0 + shift) * a.vT;
#pragma unroll
        for (int i = 0; i < F::KL; ++i) {
          const int s = tid + 256 * i;
          kr[i] = load_16(kp + (s / F::KCH) * a.kT + 16 * (s % F::KCH));
        }
#pragma unroll
        for (int i = 0; i < F::VL; ++i) {
          const int s = tid + 256 * i;
          vr[i] = load_16(vp + (s / F::VCH) * a.vT + 16 * (s % F::VCH));
        }
      } else {
#pragma unroll
        for (int i = 0; i < F::KL; ++i) {
          const int s = tid + 256 * i, v = v0 + s / F::KCH, c = s % F::KCH;
          kr[i] = v < nv && F::VEC * c < a.d ? load_16(kb + (int64_t)(v < ns ? v : v + shift) * a.kT + 16 * c) : zero4;
        }
#pragma unroll
        for (int i = 0; i < F::VL; ++i) {
          const int s = tid + 256 * i, v = v0 + s / F::VCH, c = s % F::VCH;
          vr[i] = v < nv && F::VEC * c < a.dv ? load_16(vb + (int64_t)(v < ns ? v : v + shift) * a.vT + 16 * c) : zero4;
        }
      }
    };
    auto store = [&](int blk) {
      char* ks = smem + (blk & 1) * (F::K_BYTES + F::V_BYTES);
#pragma unroll
      for (int i = 0; i < F::KL; ++i) {
        const int s = tid + 256 * i;
        *reinterpret_cast<u32x4_t*>(ks + F::k_off(s / F::KCH, s % F::KCH)) = kr[i];
      }
#pragma unroll
      for (int i = 0; i < F::VL; ++i) {
        const int s = tid + 256 * i;
        *reinterpret_cast<u32x4_t*>(ks + F::K_BYTES + F::v_off(s / F::VCH, F::VEC * (s % F::VCH))) = vr[i];
      }
    };

    // m: largest score so far (raw), sh = m * scale, l: this lane's part of the row's sum
    float m = -INFINITY, sh = 0.f, l = 0.f;
    f32x16_t oacc[F::OF];  // O^T: register r of block e is column 32e + 8(r/4) + 4hf + r%4 of row l32
#pragma unroll
    for (int e = 0; e < F::OF; ++e)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[e][r] = 0.f;

    auto block = [&](int blk, auto open) {
      const char* ks = smem + (blk & 1) * (F::K_BYTES + F::V_BYTES);
      const char* vs = ks + F::K_BYTES;
      f32x16_t sc[NH];
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[hb][r] = 0.f;
#pragma unroll
        for (int c = 0; c < F::QF; ++c)
          Mfma<T>::step(sc[hb], *reinterpret_cast<const u32x4_t*>(ks + F::k_off(32 * hb + l32, 2 * c + hf)), qf[c]);
      }
      if constexpr (!decltype(open)::value) {
#pragma unroll
        for (int hb = 0; hb < NH; ++hb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int v = blk * BN + 32 * hb + 8 * (r >> 2) + 4 * hf + (r & 3);
            const int key = v < ns ? v : v + shift;
            const bool seen = row_ok && v < nv && key <= p && (p - key < a.window || key < a.sinks);
            sc[hb][r] = seen ? sc[hb][r] : -INFINITY;
          }
      }
      float mx = sc[0][0];
#pragma unroll
      for (int hb = 0; hb < NH; ++hb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[hb][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float to = mn == -INFINITY ? 0.f : mn * a.scale;
        const float corr = mx > m ? (m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sh - to)) : 1.f;
        l *= corr;
#pragma unroll
        for (int e = 0; e < F::OF; ++e)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[e][r] *= corr;
        m = mn;
        sh = to;
      }
#pragma unroll
      for (int hb = 0; hb < NH; ++hb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sc[hb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[hb][r], a.scale, -sh));
          l += sc[hb][r];
        }
        if constexpr (E == 4) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int e = 0; e < F::OF; ++e)
              oacc[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                  *reinterpret_cast<const float*>(vs + F::v_off(32 * hb + 8 * (r >> 2) + 4 * hf + (r & 3), 32 * e + l32)),
                  sc[hb][r], oacc[e], 0, 0, 0);
        } else {
          // transposing reads: lane s of a 16-lane group points at row k0 + s/4, column n0 + 4(s%4), and
          // receives rows k0 .. k0+3 of column n0 + s
          const int vrow = 4 * hf + ((lane & 15) >> 2), vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2) {
            u32x4_t pb;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = sc[hb][8 * c2 + 2 * i], y = sc[hb][8 * c2 + 2 * i + 1];
              if constexpr (std::is_same<T, bf16_t>::value) pb[i] = f32x2_to_bf16x2_bits(x, y);
              else pb[i] = (uint32_t)f32_to_f16_bits(x) | ((uint32_t)f32_to_f16_bits(y) << 16);
            }
            const int row = 32 * hb + 16 * c2 + vrow;
#pragma unroll
            for (int e = 0; e < F::OF; ++e) {
              const u32x2_t lo = lds_read_tr16(vs + F::v_off(row, 32 * e + vcol));
              const u32x2_t hi = lds_read_tr16(vs + F::v_off(row + 8, 32 * e + vcol));
              Mfma<T>::step(oacc[e], u32x4_t{lo[0], lo[1], hi[0], hi[1]}, pb);
            }
          }
        }
      }
    };

    if (nblk > 0) {
      load(0);
      store(0);
    }
    __syncthreads();
    for (int blk = 0; blk < nblk; ++blk) {
      if (blk + 1 < nblk) load(blk + 1);
      const int v0 = blk * BN, v1 = v0 + BN - 1;
      const int k0 = v0 < ns ? v0 : v0 + shift, k1 = v1 < ns ? v1 : v1 + shift;  // first and last key
      // any row of the wavefront sees a key / all rows see all of them
      const bool some = 32 * w < qrows && k0 <= wp1 && (v0 < ns || k0 < a.sinks || (int64_t)k1 > (int64_t)wp0 - a.window);
      const bool all = 32 * w + 31 < qrows && v1 < nv && k1 <= wp0 && v0 >= ns && (int64_t)wp1 - k0 < a.window;
      if (all) block(blk, std::true_type{});
      else if (some) block(blk, std::false_type{});
      if (blk + 1 < nblk) store(blk + 1);
      __syncthreads();
    }

    l += __shfl_xor(l, 32, 64);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bool lost = false;  // an output that is not finite over a finite sum
    if (l > 0.f && l < INFINITY) {
#pragma unroll
      for (int e = 0; e < F::OF; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r) lost |= !(fabsf(oacc[e][r]) < INFINITY);
    }
    const uint64_t again = __ballot(lost && row_ok);
    const bool mine_again = (again >> l32 | again >> (l32 + 32)) & 1;
    if (row_ok && !mine_again) {
      char* orow = ob + rloc * a.oT;
#pragma unroll
      for (int e = 0; e < F::OF; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = 32 * e + 8 * j + 4 * hf;
          if (col >= a.dv) continue;
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = l == 0.f ? 0.f : oacc[e][4 * j + i] * inv;
          if constexpr (E == 4) {
            *reinterpret_cast<u32x4_any_t*>(orow + E * col) =
                u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
          } else if constexpr (std::is_same<T, bf16_t>::value) {
            *reinterpret_cast<u32x2_any_t*>(orow + E * col) = u32x2_t{f32x2_to_bf16x2_bits(x[0], x[1]), f32x2_to_bf16x2_bits(x[2], x[3])};
          } else {
            *reinterpret_cast<u32x2_any_t*>(orow + E * col) =
                u32x2_t{(uint32_t)f32_to_f16_bits(x[0]) | ((uint32_t)f32_to_f16_bits(x[1]) << 16),
                        (uint32_t)f32_to_f16_bits(x[2]) | ((uint32_t)f32_to_f16_bits(x[3]) << 16)};
          }
        }
    }
    for (uint64_t rest = (again | again >> 32) & 0xffffffffull; rest != 0; rest &= rest - 1) {
      const int r = 32 * w + __builtin_ctzll(rest);
      window_row<T>(a, qb + r * a.qT, kb, vb, ob + r * a.oT, p0 + r, kl, lane);
    }
  }
}

template <typename T, int DP, int DVP>
static int window_launch(const WindowArgs& a, hipStream_t s) {
  const int64_t most = 1 << 22;  // a multiple of kWindowOrder; further tiles by the kernel's own loop
  hipLaunchKernelGGL((window_attn_kernel<T, DP, DVP>), dim3((unsigned)(a.total < most ? a.total : most)), dim3(256), 0, s, a);
  return check_launch("window_attn_kernel");
}
template <typename T>
static int window_launch_d(const WindowArgs& a, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (a.d > 128 || a.dv > 128) return window_launch<T, 256, 256>(a, s);
  }
  if (a.d <= 64 && a.dv <= 64) return window_launch<T, 64, 64>(a, s);
  return window_launch<T, 128, 128>(a, s);
}

}  // namespace biops

using namespace biops;

extern "C" int biops_window_attention_max_head(int dtype) {
  return dtype == BIOPS_F32 ? 128 : (dtype == BIOPS_F16 || dtype == BIOPS_BF16 ? 256 : 0);
}

extern "C" int biops_window_attention(int dtype, int64_t nseq, int64_t hq, int64_t hkv, int64_t lq, int64_t lk, int64_t d,
                                      int64_t dv, const void* q, int64_t sqB, int64_t sqT, int64_t sqH, const void* k,
                                      int64_t skB, int64_t skT, int64_t skH, const void* v, int64_t svB, int64_t svT,
                                      int64_t svH, void* out, int64_t soB, int64_t soT, int64_t soH, const void* cu_q,
                                      int cu_q64, int64_t cu_q_stride, const void* cu_k, int cu_k64, int64_t cu_k_stride,
                                      int64_t window, int64_t sinks, float scale, int* flag, void* stream) {
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
  if (hq == 0 || lq == 0 || (!cu_q && nseq == 0)) return BIOPS_OK;
  if (!q || !out || (lk > 0 && (!k || !v)) || (cu_q && (!cu_k || !flag)))
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
  a.hkv = (int)hkv, a.group = (int)(hq / hkv);
  a.d = (int)d, a.dv = (int)dv;
  const int64_t all = INT64_C(0x7fffffff);
  a.window = (int)(window < all ? window : all), a.sinks = (int)(sinks < all ? sinks : all);
  a.negate = scale < 0.f;
  // a scale of zero: every weight 1, and 0 * -inf stays out of the masked scores
  const float s = (scale < 0.f ? -scale : scale) * kLog2e;
  a.scale = s > 1e-30f ? s : 1e-30f;
  // packed: every sequence and the two ends may end in a part of a tile
  const int64_t tiles = cu_q ? lq / kWindowRows + nseq + 2 : cdiv(lq, kWindowRows);
  if (tiles > all) return fail(BIOPS_ERR_ARG, "biops_window_attention: too many sequences");
  a.tiles = (int)tiles;
  a.total = tiles * hq * (cu_q ? 1 : nseq);
  BIOPS_DISPATCH_FLOAT(dtype, return window_launch_d<T>(a, static_cast<hipStream_t>(stream)));
  return BIOPS_OK;
}

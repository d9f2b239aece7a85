// Attention of one new token per sequence over a cache in pages whose keys and values are held in 4 bits (fp4.h).
//
// The mathematics, the chunks and the join are those of the attention over 16-bit pages (paged_attention.hip): a workgroup
// takes a chunk of a sequence's visible keys for the query heads that share a key/value head, scores and weighted sums go
// through 16x16 MFMAs, and a second kernel joins the chunks.  Here a row of keys is 17 bytes for 32 elements.  They become
// 16-bit values in registers, exactly, by one conversion for two elements that multiplies with the block's power of two too.
// The order of a key's elements inside the dot product is free, so a lane takes a whole block of a key (16 bytes, one
// exponent) where 128 elements make four of them, and the queries are laid out the same way.
//
// Exponents are read by key: lane l < 32 has those of key l of the tile, the others those of its value, and the wavefront
// exchanges them through LDS together with the rows' places.
//
// A key's 4.25 bits an element leave less to wait for than to compute: 64 sequences of 250 to 16384 keys (16/4 heads of 128,
// bf16) take 54 us and 5 for the join, 2.3 TB/s of 137 MB, where the 16-bit pages take 114 us.  Vector instructions issue in
// about half of the cycles (a value element costs half a conversion, a byte permutation and its share of two MFMAs).
// Registers for three wavefronts a SIMD are what 128-wide heads fit into; for four, they spill and it is slower.  Values are
// converted four columns at a time for the same reason.  One sequence of 2047 keys: 6.4 us, and 3.8 for the join, bound by
// three reads that wait for one another (length, pages, rows).
#include "fp4.h"
#include "paged_attention.h"

namespace biops {

struct Paged4Args : PagedArgs {
  const char *ks, *vs;                       // exponents
  int64_t ksP, ksS, ksH, vsP, vsS, vsH;      // byte strides
  uint32_t page_factor, page_shift;          // key / page_size = key page_factor >> page_shift
};

typedef u32x4_t u32x4_byte_t __attribute__((aligned(1)));
typedef u32x2_t u32x2_byte_t __attribute__((aligned(1)));
typedef uint32_t u32_byte_t __attribute__((aligned(1)));
typedef uint16_t u16_byte_t __attribute__((aligned(1)));

constexpr float kSlack = 8.f;  // powers of two that a weight may be larger than 1

// Wavefronts per SIMD that registers are given out for.
template <int DP, int DVP>
constexpr int paged4_waves() {
  constexpr int wide = DP > DVP ? DP : DVP;
  return wide <= 64 ? 4 : (wide <= 128 ? 3 : 2);
}

// WHOLE: the head sizes are DP and DVP (and no lane is without elements).
template <typename T, int DP, int DVP, bool WHOLE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(paged4_waves<DP, DVP>(), paged4_waves<DP, DVP>())))
void paged4_chunk_kernel(Paged4Args a) {
  constexpr int KB = DP <= 64 ? 1 : DP / 128;           // blocks (or halves of one) of a key that a lane has
  constexpr int KW = DP <= 64 ? 2 : 4;                  // their dwords
  constexpr int KS = KB * KW;                           // score steps: 8 elements of each of the four lanes of a key
  constexpr int W = DVP <= 64 ? 4 : 8;                  // elements of a value load
  constexpr int NB = DVP / (16 * W), NT = NB * W;       // value loads of a row; 16-column output blocks
  constexpr int XW = DP > 128 || DVP > 128 ? 2 : 1;     // dwords of a row's exponents
  extern __shared__ __attribute__((aligned(16))) char smem[];  // as paged_finish has it
  __shared__ __attribute__((aligned(16))) int64_t offs[4][2][32];
  __shared__ __attribute__((aligned(16))) uint32_t exps[4][XW][2][32];
  __shared__ int bad_page;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int m16 = lane & 15, q4 = lane >> 4;
  const int64_t heads = (int64_t)a.hkv * a.group;

  // Workgroups go round over the eight XCDs: the heads of a chunk, whose rows share lines of memory, to the same one.
  const uint32_t across = a.hkv * a.zs, id = a.first + blockIdx.x;
  const uint32_t r = (id >> 3) % across;
  const uint32_t z = r % a.zs, hk = r / a.zs;
  uint32_t b = 8 * ((id >> 3) / across) + (id & 7);
  int c = 0, length;
  if (a.chunks == 1) {
    if (b >= a.batch) return;
    length = paged_length(a, b);
  } else if (a.batch <= kPagedListed) {
    if (!paged_find(a, (int)b, lane, b, c, length)) return;
  } else {  // first chunks of all sequences, then second ones: what is idle comes last
    c = (int)(b / a.batch);
    b -= c * a.batch;
    if (c >= a.chunks) return;
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

  // first element of this lane's score step s
  auto element = [&](int s) { return DP <= 64 ? 16 * q4 + 8 * s : 128 * (s >> 2) + 32 * q4 + 8 * (s & 3); };
  u32x4_t qf[KS];  // queries (B operand): column m16
  {
    const char* qr = a.q + b * a.qB + (h0 + (m16 < cols ? m16 : 0)) * a.qH;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = element(s);
      qf[s] = m16 < cols && (WHOLE || d0 < a.d) ? load_16(qr + 2 * d0) : u32x4_t{0u, 0u, 0u, 0u};
      if (a.negate | a.zero) qf[s] = score_query<T>(qf[s], a.negate, a.zero);
    }
  }
  __syncthreads();  // bad_page is clear

  // Key `lane % 32` of a tile: its page, then the byte offset of its keys (lanes 0-31) or values, and their exponents (1
  // behind the end).
  const bool is_key = lane < 32;
  const int blocks = (is_key ? a.d : a.dv) >> 5;
  const int64_t rowP = is_key ? a.kP : a.vP, rowS = is_key ? a.kS : a.vS;
  const int64_t expP = is_key ? a.ksP : a.vsP, expS = is_key ? a.ksS : a.vsS;
  const char* const eb = is_key ? a.ks + hk * a.ksH : a.vs + hk * a.vsH;
  auto key_at = [&](int tile) {
    const int i = 32 * tile + (lane & 31), v = v0 + (i < nkeys ? i : nkeys - 1);
    return (uint32_t)(v < span.ns ? v : v + span.shift);
  };
  auto page_of = [&](int tile) -> int64_t {
    const int64_t e = b * a.tB + (uint32_t)((uint64_t)key_at(tile) * a.page_factor >> a.page_shift) * a.tW;
    return a.table64 ? reinterpret_cast<const int64_t*>(a.table)[e] : (int64_t) reinterpret_cast<const int32_t*>(a.table)[e];
  };
  struct Exps {
    uint32_t word[XW];
  };
  bool bad = false;

  struct Tile {
    uint32_t k[2][KB][KW];
    uint32_t v[NB][8];
  };
  const char* const kb = a.kc + hk * a.kH;
  const char* const vb = a.vc + hk * a.vH;
  // the loads of a tile whose pages are `id`
  auto fetch = [&](Tile& t, Exps& x, int tile, int64_t id) {
    if (id < 0 || id >= a.pages) {
      bad = true;
      id = 0;
    }
    const uint32_t key = key_at(tile), at = key - (uint32_t)((uint64_t)key * a.page_factor >> a.page_shift) * a.page_size;
    offs[w][lane >> 5][lane & 31] = id * rowP + at * rowS;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const char* e = eb + id * expP + at * expS;
    if constexpr (WHOLE && DP == 128 && DVP == 128) {
      x.word[0] = *reinterpret_cast<const u32_byte_t*>(e);
    } else {
#pragma unroll
      for (int j = 0; j < XW; ++j) x.word[j] = 0x7f7f7f7fu;
#pragma unroll
      for (int j = 0; j < (DP > DVP ? DP : DVP) / 32; ++j)
        if ((WHOLE && DP == DVP) || j < blocks) x.word[j >> 2] = (x.word[j >> 2] & ~(255u << (8 * (j & 3)))) | (uint32_t)(uint8_t)e[j] << (8 * (j & 3));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* p = kb + offs[w][0][8 * (m16 >> 2) + 4 * i + (m16 & 3)];
#pragma unroll
      for (int s = 0; s < KB; ++s) {
        const int d0 = element(s * KW);
        if constexpr (KW == 4) {
          const u32x4_t x = WHOLE || d0 < a.d ? u32x4_t(*reinterpret_cast<const u32x4_byte_t*>(p + (d0 >> 1))) : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
          for (int j = 0; j < 4; ++j) t.k[i][s][j] = x[j];
        } else {
          const u32x2_t x = WHOLE || d0 < a.d ? u32x2_t(*reinterpret_cast<const u32x2_byte_t*>(p + (d0 >> 1))) : u32x2_t{0u, 0u};
          t.k[i][s][0] = x[0];
          t.k[i][s][1] = x[1];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* p = vb + offs[w][1][8 * q4 + j];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int e0 = 16 * W * n + W * m16;
        if constexpr (W == 8) t.v[n][j] = WHOLE || e0 < a.dv ? *reinterpret_cast<const u32_byte_t*>(p + (e0 >> 1)) : 0u;
        else t.v[n][j] = WHOLE || e0 < a.dv ? (uint32_t)*reinterpret_cast<const u16_byte_t*>(p + (e0 >> 1)) : 0u;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  // byte `at` of a word in the place of a float's exponent
  auto power = [](uint32_t word, int at) {
    return __uint_as_float(__builtin_amdgcn_alignbit(word, word, (8 * at + 9) & 31) & 0x7f800000u);
  };

  // of query m16: largest product so far, the same or 0 where that is -inf, sum (of this lane's keys)
  float m, from, l;
  f32x4_t acc[NT];
  float down = -kPagedUp<T>;  // powers of two that are off the weights
  for (;;) {
    m = -INFINITY, from = 0.f, l = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // One wait a tile: while it is worked on, the next one's rows and the pages of the one after it are on their way.
    Tile cur, next;
    Exps here, there;
    int64_t id = 0;
    if (w < tiles) {
      fetch(cur, here, w, page_of(w));
      if (w + 4 < tiles) id = page_of(w + 4);
    }
    for (int tile = w; tile < tiles; tile += 4) {
      if (32 * tile + (lane & 31) >= nkeys)
#pragma unroll
        for (int j = 0; j < XW; ++j) here.word[j] = 0x7f7f7f7fu;
#pragma unroll
      for (int j = 0; j < XW; ++j) exps[w][j][lane >> 5][lane & 31] = here.word[j];
      if (tile + 4 < tiles) {
        fetch(next, there, tile + 4, id);
        if (tile + 8 < tiles) id = page_of(tile + 8);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      f32x4_t sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KB; ++s) {
          const float x = power(exps[w][s][0][8 * (m16 >> 2) + 4 * i + (m16 & 3)], KW == 4 ? q4 : q4 >> 1);
#pragma unroll
          for (int j = 0; j < KW; ++j) mfma16<T>(sc[i], fp4_values<T>(cur.k[i][s][j], x), qf[s * KW + j]);
        }
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
          for (int n = 0; n < NB; ++n) cur.v[n][j] = in ? cur.v[n][j] : 0u;
        }
      }
      float mx = p[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, p[j]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      // The sums are rescaled where a product has grown past the last maximum by 2^kSlack in its weight: weights go up to that.
      if (__any((mx - m) * a.scale > kSlack || (mx > m && m == -INFINITY))) {
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
      u32x4_t hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hi[i] = pack_pair<T>(p[2 * i], p[2 * i + 1]);
        lo[i] = pack_pair<T>(p[2 * i] - Num<T>::from_bits(hi[i] & 0xffffu), p[2 * i + 1] - Num<T>::from_bits(hi[i] >> 16));
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float power_of[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) power_of[j] = power(exps[w][n][1][8 * q4 + j], W == 8 ? m16 >> 2 : m16 >> 3);
        // four columns of value rows 8 q4 .. 8 q4 + 7 at a time (all eight take registers of a whole wavefront)
        auto columns = [&](auto half) {
          constexpr int H = decltype(half)::value;
          uint32_t rows[8][2];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            rows[j][0] = fp4_pair<T, 2 * H>(cur.v[n][j], power_of[j]);
            rows[j][1] = fp4_pair<T, 2 * H + 1>(cur.v[n][j], power_of[j]);
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            u32x4_t va;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              va[i] = __builtin_amdgcn_perm(rows[2 * i + 1][t >> 1], rows[2 * i][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            mfma16<T>(acc[W * n + 4 * H + t], va, hi);
            mfma16<T>(acc[W * n + 4 * H + t], va, lo);
          }
        };
        columns(std::integral_constant<int, 0>());
        if constexpr (W == 8) {
          __builtin_amdgcn_sched_barrier(0);
          columns(std::integral_constant<int, 1>());
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      cur = next;
      here = there;
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
    if (past) down = kSlack + (float)(32 - __builtin_clz((uint32_t)span.chunk / 4));  // (a wavefront has a quarter of the chunk's keys)
  }
  paged_finish<T, DVP, W>(a, smem, &bad_page, m, l, down, bad, acc, b, h0, c, cols);
}

template <typename T, int DP, int DVP>
static int paged4_launch(Paged4Args a, hipStream_t s) {
  const unsigned cols = a.group < kPagedCols ? a.group : kPagedCols;
  const unsigned lds = (unsigned)(4 * cols * (DVP + 2) * sizeof(float));
  constexpr uint32_t most = 1 << 22;  // a launch has less than 2^32 threads
  const uint32_t items = a.batch * a.chunks;
  const uint32_t total = ((items + 7) & ~7u) * (a.hkv * a.zs);
  for (a.first = 0; a.first < total; a.first += most) {
    const uint32_t n = total - a.first < most ? total - a.first : most;
    if (a.d == DP && a.dv == DVP) hipLaunchKernelGGL((paged4_chunk_kernel<T, DP, DVP, true>), dim3(n), dim3(256), lds, s, a);
    else hipLaunchKernelGGL((paged4_chunk_kernel<T, DP, DVP, false>), dim3(n), dim3(256), lds, s, a);
    const int rc = check_launch("paged4_chunk_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  return paged_join<T>(a, s);
}
template <typename T, int DP>
static int paged4_launch_dv(const Paged4Args& a, hipStream_t s) {
  if (a.dv <= 64) return paged4_launch<T, DP, 64>(a, s);
  if (a.dv <= 128) return paged4_launch<T, DP, 128>(a, s);
  return paged4_launch<T, DP, 256>(a, s);
}
template <typename T>
static int paged4_launch_d(const Paged4Args& a, hipStream_t s) {
  if (a.d <= 64) return paged4_launch_dv<T, 64>(a, s);
  if (a.d <= 128) return paged4_launch_dv<T, 128>(a, s);
  return paged4_launch_dv<T, 256>(a, s);
}

}  // namespace biops

using namespace biops;

extern "C" int biops_paged_attention_fp4(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t dv,
                                         const void* q, int64_t sqB, int64_t sqH, const void* kc, int64_t skP, int64_t skS,
                                         int64_t skH, const void* ks, int64_t sksP, int64_t sksS, int64_t sksH, const void* vc,
                                         int64_t svP, int64_t svS, int64_t svH, const void* vs, int64_t svsP, int64_t svsS,
                                         int64_t svsH, int64_t pages, int64_t page_size, const void* table, int table64,
                                         int64_t stB, int64_t stW, int64_t width, const void* lengths, int lengths64,
                                         int64_t slB, int64_t max_length, int64_t window, int64_t sinks, float scale,
                                         void* out, int* flag, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != BIOPS_F16 && dtype != BIOPS_BF16) return fail(BIOPS_ERR_DTYPE, "biops_paged_attention_fp4: unsupported dtype %d", dtype);
  if (batch < 0 || hq < 0 || hkv <= 0 || hq % hkv != 0) return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: bad batch or heads");
  if (d < kFp4Block || d > 256 || d % kFp4Block || dv < kFp4Block || dv > 256 || dv % kFp4Block)
    return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: head sizes are multiples of %d up to 256", kFp4Block);
  if (pages <= 0 || page_size <= 0 || width < 0 || page_size > INT64_C(0x7fffffff))
    return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: a cache without pages");
  if (window < 0 || sinks < 0) return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: negative window");
  if (!(scale - scale == 0.f)) return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: scale is not finite");
  if (batch == 0 || hq == 0) return BIOPS_OK;
  if (!q || !kc || !ks || !vc || !vs || !lengths || !out || !flag || (width > 0 && !table))
    return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: null pointer");
  // counted in 32 bits: workgroups and output rows
  if (hq > (INT64_C(1) << 30) / kPagedChunks / batch) return fail(BIOPS_ERR_ARG, "biops_paged_attention_fp4: more than 2^24 rows");
  Paged4Args a;
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
      return fail(BIOPS_ERR_SIZE, "biops_paged_attention_fp4: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BIOPS_ERR_LAYOUT, "biops_paged_attention_fp4: workspace not 16-byte aligned");
  }
  a.part = static_cast<float*>(workspace);
  a.ml = a.part + rows * dv;
  a.q = static_cast<const char*>(q), a.kc = static_cast<const char*>(kc), a.vc = static_cast<const char*>(vc);
  a.ks = static_cast<const char*>(ks), a.vs = static_cast<const char*>(vs);
  a.out = static_cast<char*>(out);
  a.table = table, a.lengths = lengths, a.flag = flag;
  a.qB = 2 * sqB, a.qH = 2 * sqH;
  a.kP = skP, a.kS = skS, a.kH = skH, a.vP = svP, a.vS = svS, a.vH = svH;
  a.ksP = sksP, a.ksS = sksS, a.ksH = sksH, a.vsP = svsP, a.vsS = svsS, a.vsH = svsH;
  a.tB = stB, a.tW = stW, a.lB = slB;
  a.pages = pages, a.page_size = (uint32_t)page_size;
  a.d = (int)d, a.dv = (int)dv;
  // keys are below 2^31: with 2^l >= page_size the factor floor(2^(31 + l) / page_size) + 1 is off by at most 2^l / 2^(31 + l)
  int bits = 0;
  while ((INT64_C(1) << bits) < page_size) ++bits;
  a.page_shift = 31 + bits;
  a.page_factor = (uint32_t)((UINT64_C(1) << a.page_shift) / (uint64_t)page_size + 1);
  a.window = (int)(window < all ? window : all), a.sinks = (int)(sinks < all ? sinks : all);
  a.table64 = table64 != 0, a.lengths64 = lengths64 != 0;
  a.scale = score_scale(scale, &a.negate, &a.zero);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == BIOPS_F16) return paged4_launch_d<f16_t>(a, s);
  return paged4_launch_d<bf16_t>(a, s);
}

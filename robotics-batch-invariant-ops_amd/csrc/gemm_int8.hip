// Linear layers of 8-bit integers: rows quantised with a step of their own, and their product with a weight that has a step
// for each output channel.
//
// quantise: s_m = max_k |x_mk| / 127, q_mk = the nearest integer to x_mk (127 / max), in 32-bit arithmetic, ties to even.
// product:  y_mn = (sum_k q_mk w_nk) s_m t_n + b_n: integer sums of 32 bits, which are exact and the same in any order (up to
// 131071 terms), then 32-bit floats and one rounding.
//
// Few rows: the weight's stream from memory bounds it.  A workgroup takes 16 columns for all rows, its wavefronts parts of K;
// rows of both operands go straight to registers in the order that v_mfma_i32_16x16x64_i8 takes (any order will do that is
// the same for both), and the parts meet in LDS.  Many rows: the matrix cores bound it.  The blocks and the schedule
// are those of the 16-bit products (gemm_big.h) with twice the elements to a byte; K off the 128-byte step, or rows off 16
// bytes, go through registers in 64 x 64 blocks instead.
//
// 16 x 2048 -> 8192 takes 7.1 us, 2.4 TB/s of the weight (from the caches where they hold it); 4096 x 8192 -> 2048 65 to 70 us, 2.0 to
// 2.1 Pop/s, where the library's product of 8192^3 reaches 2.1; 777 x 2050 -> 1031 11.9 to 15.7 us by machine.  Quantising reads a row once (its elements stay in
// registers up to 8192 of them): 4096 x 8192 in bf16 20 to 23 us, 4.4 to 5 TB/s.
#include "gemm_big.h"

namespace biops {

struct i8_t { int8_t v; };
typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
typedef int32_t i32x16_t __attribute__((ext_vector_type(16)));
template <> struct Mfma<i8_t> {
  typedef i32x16_t Acc;
  __device__ static __forceinline__ void step(i32x16_t& acc, const u32x4_t& a, const u32x4_t& b) {
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), acc, 0, 0, 0);
  }
};

typedef u32x4_t u32x4_byte_t __attribute__((aligned(1)));
typedef u32x2_t u32x2_byte_t __attribute__((aligned(1)));

// ------------------------------------------------------------------------------- quantise ----
struct QuantArgs {
  const char* x;
  int8_t* q;
  float* scale;
  int64_t ld;    // bytes between rows
  int64_t rows;
  int k;
};

template <typename T>
__device__ __forceinline__ void eight_values(const T* row, int i, int k, float (&x)[8]) {
  if (i + 8 <= k) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
      const u32x4_t v = load_16(row + i + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) x[4 * h + j] = __uint_as_float(v[j]);
        else {
          x[2 * j] = Num<T>::from_bits(v[j] & 0xffffu);
          x[2 * j + 1] = Num<T>::from_bits(v[j] >> 16);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < k ? Num<T>::load(row + i + j) : 0.f;
  }
}

// THREADS of a row (64: four rows a workgroup); a thread keeps its first KEEP eights in registers and reads further ones twice.
template <typename T, int THREADS>
__global__ __launch_bounds__(256) void quantize_kernel(QuantArgs a) {
  constexpr int KEEP = 4, ROWS = 256 / THREADS;
  __shared__ uint32_t tops[4];
  const int tid = threadIdx.x % THREADS;
  const int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (THREADS == 64 && r >= a.rows) return;
  const T* row = reinterpret_cast<const T*>(a.x + r * a.ld);
  float x[KEEP][8];
  uint32_t top = 0u;
  auto look = [&](const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
      top = b > top ? b : top;
    }
  };
#pragma unroll
  for (int c = 0; c < KEEP; ++c)
    if (8 * (tid + THREADS * c) < a.k) {
      eight_values<T>(row, 8 * (tid + THREADS * c), a.k, x[c]);
      look(x[c]);
    }
  for (int i = 8 * (tid + THREADS * KEEP); i < a.k; i += 8 * THREADS) {
    float v[8];
    eight_values<T>(row, i, a.k, v);
    look(v);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t b = (uint32_t)__shfl_xor((int)top, o, 64);
    top = b > top ? b : top;
  }
  if constexpr (THREADS == 256) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
  }
  // (steps of tiny rows, and 127 / max, stay normal numbers: a row below 2^-100 keeps a step of 2^-100 / 127)
  const bool finite = top < 0x7f800000u;
  const float most = fmaxf(__uint_as_float(top), 0x1p-100f);
  const float inverse = 127.f / most;
  if (tid == 0) a.scale[r] = finite ? most / 127.f : __uint_as_float(0x7fc00000u);
  int8_t* const out = a.q + r * a.k;
  auto put = [&](const float (&v)[8], int i) {
    uint32_t b[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = finite ? (int)rintf(v[j] * inverse) : 0;
      b[j >> 2] |= ((uint32_t)n & 255u) << (8 * (j & 3));
    }
    if (i + 8 <= a.k) {
      *reinterpret_cast<u32x2_byte_t*>(out + i) = u32x2_t{b[0], b[1]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < a.k) out[i + j] = (int8_t)(b[j >> 2] >> (8 * (j & 3)));
    }
  };
#pragma unroll
  for (int c = 0; c < KEEP; ++c)
    if (8 * (tid + THREADS * c) < a.k) put(x[c], 8 * (tid + THREADS * c));
  for (int i = 8 * (tid + THREADS * KEEP); i < a.k; i += 8 * THREADS) {
    float v[8];
    eight_values<T>(row, i, a.k, v);
    put(v, i);
  }
}

template <typename T>
static int quantize_launch(const QuantArgs& a, hipStream_t s) {
  if (a.k <= 1024) hipLaunchKernelGGL((quantize_kernel<T, 64>), dim3((unsigned)cdiv(a.rows, 4)), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quantize_kernel<T, 256>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
  return check_launch("quantize_kernel");
}

// -------------------------------------------------------------------------------- product ----
struct Int8Args {
  const int8_t *x, *w;
  const float *xs, *ws;
  const void* bias;
  void* y;
  int64_t ldx, ldw;          // bytes between rows
  int64_t xs_s, ws_s;
  int64_t M, N, K;
  int tiles_m, tiles_n, total;
  int nt;                    // non-temporal stores (gemm_big.h)
};

// The first product, sums of up to 2^31 times a row's step, is past 32-bit floats from a step of 2^97 on, whatever the result is.
__device__ __forceinline__ bool far_step(float xs) { return fabsf(xs) >= 0x1p96f && fabsf(xs) < INFINITY; }
// FAR: there may be such steps.  2^64 of them go to the channel's scale, exactly: what was in range has the same bits.
template <bool FAR>
__device__ __forceinline__ float finished(int32_t acc, float xs, float ws, float bias) {
  if constexpr (FAR) {
    const bool far = acc != 0 && far_step(xs);
    xs = far ? xs * 0x1p-64f : xs;
    ws = far ? ws * 0x1p64f : ws;
  }
  return __builtin_fmaf((float)acc * xs, ws, bias);
}

template <typename T, bool NT>
__device__ __forceinline__ void put_value(T* p, float v) {
  if constexpr (NT && sizeof(T) == 2) __builtin_nontemporal_store(Num<T>::to_bits(v), reinterpret_cast<uint16_t*>(p));
  else Num<T>::store(p, v);
}

// 16 bytes of a row from byte k on; zeros from byte K on.  (The last ones come as the row's last 16, shifted: byte for byte they
// took a fifth of the time of 3000 x 4001 x 1032.)
__device__ __forceinline__ u32x4_t row_bytes(const int8_t* row, int64_t k, int64_t K) {
  if (k + 16 <= K) return *reinterpret_cast<const u32x4_byte_t*>(row + k);
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (k >= K) return v;
  if (K < 16) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (k + j < K) v[j >> 2] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j & 3));
    return v;
  }
  v = *reinterpret_cast<const u32x4_byte_t*>(row + K - 16);
  const int by = 8 * (int)(16 - (K - k));  // 8 .. 120
  const uint64_t low = (uint64_t)v[1] << 32 | v[0], high = (uint64_t)v[3] << 32 | v[2];
  const uint64_t first = by < 64 ? low >> by | high << (64 - by) : high >> (by - 64), second = by < 64 ? high >> by : 0u;
  return u32x4_t{(uint32_t)first, (uint32_t)(first >> 32), (uint32_t)second, (uint32_t)(second >> 32)};
}

// MB blocks of 16 rows; WAVES wavefronts share K.
template <typename T, int MB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void int8_few_kernel(Int8Args a) {
  __shared__ __attribute__((aligned(16))) i32x4_t part[WAVES][MB][64];
  constexpr int AHEAD = 8 / MB < 2 ? 2 : 8 / MB;  // K steps of 64 bytes whose loads go out together
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, m16 = lane & 15, q4 = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + m16 < a.N ? n0 + m16 : a.N - 1;  // (rows past the end are read again and not stored)
  const int8_t* const wr = a.w + n * a.ldw;
  const int8_t* xr[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t m = 16 * i + m16 < a.M ? 16 * i + m16 : a.M - 1;
    xr[i] = a.x + m * a.ldx;
  }
  i32x4_t acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = i32x4_t{0, 0, 0, 0};
  const int64_t steps = a.K / 64, per = (steps + WAVES - 1) / WAVES;  // whole steps, of 64 bytes
  const int64_t s1 = (w + 1) * per < steps ? (w + 1) * per : steps;
  auto product = [&](const u32x4_t& b, const u32x4_t (&x)[MB]) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
      acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, x[i]), __builtin_bit_cast(i32x4_t, b), acc[i], 0, 0, 0);
  };
  for (int64_t s = w * per; s < s1; s += AHEAD) {
    u32x4_t b[AHEAD], x[AHEAD][MB];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (s + j >= s1) break;
      const int64_t k = 64 * (s + j) + 16 * q4;
      b[j] = *reinterpret_cast<const u32x4_byte_t*>(wr + k);
#pragma unroll
      for (int i = 0; i < MB; ++i) x[j][i] = *reinterpret_cast<const u32x4_byte_t*>(xr[i] + k);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (s + j >= s1) break;
      product(b[j], x[j]);
    }
  }
  if (w == WAVES - 1 && a.K % 64 != 0) {
    const int64_t k = 64 * steps + 16 * q4;
    u32x4_t x[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) x[i] = row_bytes(xr[i], k, a.K);
    product(row_bytes(wr, k, a.K), x);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) part[w][i][lane] = acc[i];
  __syncthreads();
  for (int u = tid; u < MB * 64; u += 64 * WAVES) {
    const int i = u >> 6, l = u & 63;
    i32x4_t sum = part[0][i][l];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum += part[v][i][l];
    const int64_t col = n0 + (l & 15);
    if (col >= a.N) continue;
    const float ws = a.ws[col * a.ws_s], bias = a.bias ? Num<T>::load(static_cast<const T*>(a.bias) + col) : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = 16 * i + 4 * (l >> 4) + j;
      if (m < a.M) Num<T>::store(static_cast<T*>(a.y) + m * a.N + col, finished<true>(sum[j], a.xs[m * a.xs_s], ws, bias));
    }
  }
}

// Where block t of a launch begins: 8 rows of blocks are walked column by column, neighbours on one XCD.
__device__ __forceinline__ bool int8_origin(const Int8Args& a, int BM, int BN, int64_t& m0, int64_t& n0) {
  const int64_t t = xcd_slot(blockIdx.x, gridDim.x);
  if (t >= a.total) return false;
  tile_coords(t, a.tiles_m, a.tiles_n, m0, n0);
  m0 *= BM;
  n0 *= BN;
  return true;
}

template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void int8_big_kernel(Int8Args a) {
  using Tile = BigTile<i8_t, BM, BN, 128>;
  __shared__ __attribute__((aligned(16))) char smem[Tile::SMEM_BYTES];
  int64_t m0, n0;
  if (!int8_origin(a, BM, BN, m0, n0)) return;
  const int rows = a.M - m0 < BM ? (int)(a.M - m0) : BM, cols = a.N - n0 < BN ? (int)(a.N - n0) : BN;
  typename Tile::Acc acc[Tile::FM][Tile::FN];
  Tile::mainloop(smem, acc, reinterpret_cast<const i8_t*>(a.x) + m0 * a.ldx, a.ldx, rows,
                 reinterpret_cast<const i8_t*>(a.w) + n0 * a.ldw, a.ldw, cols, a.K);
  float* const xs = reinterpret_cast<float*>(smem);  // the ring is idle
  for (int i = threadIdx.x; i < BM; i += 256) xs[i] = a.xs[(m0 + (i < rows ? i : rows - 1)) * a.xs_s];
  __syncthreads();
  bool far = false;  // a row of this wavefront has such a step: it has a store of its own
  for (int i = threadIdx.x & 63; i < Tile::WM; i += 64) far |= far_step(xs[(threadIdx.x >> 7) * Tile::WM + i]);
  T* const y = static_cast<T*>(a.y) + m0 * a.N + n0;
  int ldc = (int)a.N;
  asm volatile("" : "+s"(ldc));  // (keeps the compiler from holding all row offsets)
  auto store = [&](auto checked, auto nt, auto with_far) {
#pragma unroll
    for (int j = 0; j < Tile::FN; ++j) {
      const int col = Tile::acc_col(j);
      const bool in = !checked || col < cols;
      const float ws = in ? a.ws[(n0 + col) * a.ws_s] : 0.f;
      const float bias = in && a.bias ? Num<T>::load(static_cast<const T*>(a.bias) + n0 + col) : 0.f;
#pragma unroll
      for (int i = 0; i < Tile::FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = Tile::acc_row(i, r);
          if (checked && (!in || row >= rows)) continue;
          T* const p = y + (uint32_t)(row * ldc + col);
          const float v = finished<decltype(with_far)::value>(acc[i][j][r], xs[row], ws, bias);
          put_value<T, decltype(nt)::value>(p, v);
        }
    }
  };
  const std::true_type yes;
  const std::false_type no;
  if (__any(far)) store(yes, no, yes);
  else if (rows < BM || cols < BN) store(yes, no, no);
  else if (a.nt) store(no, yes, no);
  else store(no, no, no);
}

// 64 x 64 blocks, operands through registers: any K, any alignment.
template <typename T>
__global__ __launch_bounds__(256) void int8_any_kernel(Int8Args a) {
  __shared__ __attribute__((aligned(16))) char smem[2][2][64 * 128];
  __shared__ float steps[64];
  int64_t m0, n0;
  if (!int8_origin(a, 64, 64, m0, n0)) return;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int wm = 32 * (w >> 1), wn = 32 * (w & 1), lr = lane & 31, half = lane >> 5;
  const int64_t col = n0 + wn + lr < a.N ? n0 + wn + lr : a.N - 1;
  const float ws = a.ws[col * a.ws_s], bias = a.bias ? Num<T>::load(static_cast<const T*>(a.bias) + col) : 0.f;
  if (tid < 64) steps[tid] = a.xs[(m0 + tid < a.M ? m0 + tid : a.M - 1) * a.xs_s];
  // chunk tid % 8 of rows tid / 8 and 32 further, of both operands
  const int row = tid >> 3, chunk = tid & 7;
  const int8_t *xr[2], *wr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + row + 32 * i < a.M ? m0 + row + 32 * i : a.M - 1, n = n0 + row + 32 * i < a.N ? n0 + row + 32 * i : a.N - 1;
    xr[i] = a.x + m * a.ldx;
    wr[i] = a.w + n * a.ldw;
  }
  // Whole steps: AHEAD of them are on their way.  (Loads past the last one fetch it again: issued without a condition they
  // leave the compiler a count to wait for, not all of them; 16.7 -> 14.7 us for 100 x 8000 x 2050.)
  constexpr int AHEAD = 4;
  u32x4_t x[AHEAD][2], v[AHEAD][2];
  const int64_t whole = a.K / 128;
  auto fetch = [&](int s, int64_t h) {
    const int64_t k = 128 * (h < whole ? h : whole - 1) + 16 * chunk;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[s][i] = *reinterpret_cast<const u32x4_byte_t*>(xr[i] + k);
      v[s][i] = *reinterpret_cast<const u32x4_byte_t*>(wr[i] + k);
    }
  };
  i32x16_t acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0;
  auto step = [&](int s, int buffer) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<u32x4_t*>(smem[buffer][0] + lds_off(row + 32 * i, chunk)) = x[s][i];
      *reinterpret_cast<u32x4_t*>(smem[buffer][1] + lds_off(row + 32 * i, chunk)) = v[s][i];
    }
    __syncthreads();  // (two buffers: what is written next was read before this barrier)
  };
  auto product = [&](int buffer) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      Mfma<i8_t>::step(acc, *reinterpret_cast<const u32x4_t*>(smem[buffer][0] + lds_off(wm + lr, 2 * p + half)),
                       *reinterpret_cast<const u32x4_t*>(smem[buffer][1] + lds_off(wn + lr, 2 * p + half)));
  };
  if (whole > 0) {
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) fetch(s, s);
    for (int64_t h0 = 0; h0 < whole; h0 += AHEAD)
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        if (h0 + s >= whole) break;
        step(s, s & 1);
        fetch(s, h0 + s + AHEAD);
        product(s & 1);
      }
  }
  if (a.K % 128 != 0) {
    const int64_t k = 128 * whole + 16 * chunk;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[0][i] = row_bytes(xr[i], k, a.K);
      v[0][i] = row_bytes(wr[i], k, a.K);
    }
    step(0, (int)(whole & 1));
    product((int)(whole & 1));
  }
  // The output goes through LDS for 16-byte stores: straight from the accumulators 3000 x 4001 x 136 took
  // 38.5 us, and 30.5 so.
  __syncthreads();
  T* const tile = reinterpret_cast<T*>(smem);  // [64][64]
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int m = wm + 8 * (r >> 2) + 4 * half + (r & 3);
    Num<T>::store(tile + 64 * m + wn + lr, finished<true>(acc[r], steps[m], ws, bias));
  }
  __syncthreads();
  constexpr int VEC = 16 / (int)sizeof(T), CHUNKS = 64 / VEC;
#pragma unroll
  for (int i = 0; i < 64 * CHUNKS / 256; ++i) {
    const int u = tid + 256 * i, m = u / CHUNKS, c = VEC * (u % CHUNKS);
    if (m0 + m >= a.M) continue;
    T* const to = static_cast<T*>(a.y) + (m0 + m) * a.N + n0 + c;
    if (n0 + c + VEC <= a.N) *reinterpret_cast<u32x4_any_t*>(to) = *reinterpret_cast<const u32x4_t*>(tile + 64 * m + c);
    else
      for (int e = 0; n0 + c + e < a.N; ++e) to[e] = tile[64 * m + c + e];
  }
}

template <typename T, int MB>
static int int8_few(const Int8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)cdiv(a.N, 16));
  if (a.K > 4096 && a.N <= 4096) hipLaunchKernelGGL((int8_few_kernel<T, MB, 16>), grid, dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((int8_few_kernel<T, MB, 4>), grid, dim3(256), 0, s, a);
  return check_launch("int8_few_kernel");
}
static void int8_tiles(Int8Args& a, int BM, int BN) {
  a.tiles_m = (int)cdiv(a.M, BM), a.tiles_n = (int)cdiv(a.N, BN);
  a.total = a.tiles_m * a.tiles_n;
}
template <typename T, int BM, int BN>
static int int8_big(Int8Args a, hipStream_t s) {
  int8_tiles(a, BM, BN);
  a.nt = a.total <= device_cus();
  hipLaunchKernelGGL((int8_big_kernel<T, BM, BN>), dim3((unsigned)((a.total + 7) & ~7)), dim3(256), 0, s, a);
  return check_launch("int8_big_kernel");
}
template <typename T>
static int int8_launch(Int8Args a, hipStream_t s) {
  const bool aligned = a.ldx % 16 == 0 && a.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
  const bool whole = aligned && a.K % 128 == 0;
  // Every workgroup of the kernel for few rows reads all of them, 64 bytes of a row at a time, which is slow off 16 bytes.  us (few /
  // blocks), K -> N: 2048 -> 8192 at 32 rows 9.1 / 9.5, at 64 13.2 / 8.0; 8192 -> 2048 at 32 14.2 / 19.5, at 64 21.7 / 19.3; 1024 ->
  // 1024 at 32 4.7 / 7.2; off 16 bytes 2050 -> 8000 at 16 15.9 / 11.4, 8190 -> 2040 at 16 27.9 / 28.3, at 32 40 / 28.
  // (Few columns leave few workgroups, each with all of K: the 16-bit layer of narrow blocks is then faster, 8192 -> 2048 in bf16 at
  // 32, 64 and 128 rows 11 to 15, 12 to 16 and 16 to 20 us, here 14, 19 and 19.)
  if (a.M <= 16 && (aligned || a.N <= 2048)) return int8_few<T, 1>(a, s);
  if (a.M <= 32 && aligned) return int8_few<T, 2>(a, s);
  if (whole) {
    // The blocks with the least rounds x time of a block, relative to 256 x 256.  A round of each takes, at K = 2048, 37.4 us, 23.4,
    // 14.4, 10.9 and 8.6, at K = 8192 119, 70, 41, 28 and 21.6.  (1536 x 2048 -> 6144, one round of 256 x 256 or three of 128 x 128:
    // 31.0 and 34.7 us.)
    static const struct { int bm, bn; double cost; } blocks[] = {{256, 256, 1.0}, {256, 128, 0.61}, {128, 128, 0.37}, {64, 128, 0.25}, {64, 64, 0.2}};
    const int64_t cus = device_cus();
    int best = 0;
    double least = 0.0;
    for (int i = 0; i < 5; ++i) {
      const double cost = (double)cdiv(cdiv(a.M, blocks[i].bm) * cdiv(a.N, blocks[i].bn), cus) * blocks[i].cost;
      if (i == 0 || cost < least) {
        best = i;
        least = cost;
      }
    }
    if (best == 0) return int8_big<T, 256, 256>(a, s);
    if (best == 1) return int8_big<T, 256, 128>(a, s);
    if (best == 2) return int8_big<T, 128, 128>(a, s);
    if (best == 3) return int8_big<T, 64, 128>(a, s);
    return int8_big<T, 64, 64>(a, s);
  }
  int8_tiles(a, 64, 64);
  hipLaunchKernelGGL((int8_any_kernel<T>), dim3((unsigned)((a.total + 7) & ~7)), dim3(256), 0, s, a);
  return check_launch("int8_any_kernel");
}

}  // namespace biops

using namespace biops;

extern "C" int biops_quantize_int8(int dtype, int64_t rows, int64_t k, const void* x, int64_t ld, int8_t* q, float* scale, void* stream) {
  if (!is_float_dtype(dtype)) return fail(BIOPS_ERR_DTYPE, "biops_quantize_int8: unsupported dtype %d", dtype);
  if (rows < 0 || rows > (1 << 23) || k < 1 || k > 131071) return fail(BIOPS_ERR_ARG, "biops_quantize_int8: rows of 1 to 131071 elements, at most 2^23 rows");
  if (rows == 0) return BIOPS_OK;
  if (!x || !q || !scale) return fail(BIOPS_ERR_ARG, "biops_quantize_int8: null pointer");
  QuantArgs a{static_cast<const char*>(x), q, scale, dtype_bytes(dtype) * ld, rows, (int)k};
  hipStream_t s = static_cast<hipStream_t>(stream);
  BIOPS_DISPATCH_FLOAT(dtype, return quantize_launch<T>(a, s));
  return BIOPS_OK;
}

extern "C" int biops_linear_int8(int dtype, int64_t M, int64_t N, int64_t K, const int8_t* x, int64_t ldx, const float* xs,
                                 int64_t xs_s, const int8_t* w, int64_t ldw, const float* ws, int64_t ws_s, const void* bias,
                                 void* y, void* stream) {
  if (!is_float_dtype(dtype)) return fail(BIOPS_ERR_DTYPE, "biops_linear_int8: unsupported dtype %d", dtype);
  if (M < 0 || N < 0 || K < 1 || K > 131071 || M > (1 << 23) || N > (1 << 22))
    return fail(BIOPS_ERR_ARG, "biops_linear_int8: rows of 1 to 131071 elements, at most 2^23 rows and 2^22 columns");
  if (M == 0 || N == 0) return BIOPS_OK;
  if (!x || !xs || !w || !ws || !y) return fail(BIOPS_ERR_ARG, "biops_linear_int8: null pointer");
  if (cdiv(M, 64) * cdiv(N, 64) > (1 << 23)) return fail(BIOPS_ERR_SIZE, "biops_linear_int8: too many blocks");
  Int8Args a;
  a.x = x, a.w = w, a.xs = xs, a.ws = ws, a.bias = bias, a.y = y;
  a.ldx = ldx, a.ldw = ldw, a.xs_s = xs_s, a.ws_s = ws_s;
  a.M = M, a.N = N, a.K = K, a.nt = 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  BIOPS_DISPATCH_FLOAT(dtype, return int8_launch<T>(a, s));
  return BIOPS_OK;
}

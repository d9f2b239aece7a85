// Writes rows of new keys and values into a cache in pages.
//
// Row r goes to slot s = slots[r]: page s / page_size, place s % page_size, all heads.  A negative slot
// leaves the row out (padding); a slot past the cache is left out too and reported through the flag.
// Pure data movement: each row is read and written once.
//
// Of rows that name one slot the last stays, whatever order workgroups run in: a workgroup looks
// through the slots behind its rows and leaves a row out whose slot comes again.  That is quadratic, so
// rows go in launches of kWriteRows, whose order on the stream does the rest.
#include "biops_common.h"

namespace biops {

constexpr int kWriteRows = 8192;   // rows of a launch
constexpr int kWriteGroup = 8;     // rows of a workgroup

struct WriteArgs {
  const char *k, *v;
  char *kc, *vc;
  int64_t kT, kH, vT, vH;              // byte strides of the new rows: token, head
  int64_t kcP, kcS, kcH, vcP, vcS, vcH;  // byte strides of the caches: page, slot, head
  const void* slots;
  int64_t slot_stride;
  int* flag;
  uint32_t total, page;  // slots of the cache, slots of a page
  int rows, heads, kbytes, vbytes;  // bytes of a head's row
  int slots64;
};

template <typename U>
__device__ __forceinline__ void copy_tail(const char* src, char* dst, int from, int to) {
  for (int e = from; e < to; e += sizeof(U)) *reinterpret_cast<U*>(dst + e) = *reinterpret_cast<const U*>(src + e);
}

template <int E>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
  __shared__ int64_t place[kWriteGroup];
  __shared__ int again[kWriteGroup];
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * kWriteGroup;
  const int n = a.rows - r0 < kWriteGroup ? a.rows - r0 : kWriteGroup;
  auto slot = [&](int r) -> int64_t {
    return a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[r * a.slot_stride]
                     : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[r * a.slot_stride];
  };
  if (tid < kWriteGroup) {
    int64_t s = tid < n ? slot(r0 + tid) : -1;
    if (s >= (int64_t)a.total) {
      *a.flag = 1;
      s = -1;
    }
    place[tid] = s;
    again[tid] = 0;
  }
  __syncthreads();
  int64_t mine[kWriteGroup];
#pragma unroll
  for (int i = 0; i < kWriteGroup; ++i) mine[i] = place[i];
  int hit = 0;
  for (int r = r0 + 1 + tid; r < a.rows; r += 256) {
    const int64_t s = slot(r);
#pragma unroll
    for (int i = 0; i < kWriteGroup; ++i)
      if (s == mine[i] && r > r0 + i) hit |= 1 << i;
  }
#pragma unroll
  for (int i = 0; i < kWriteGroup; ++i)
    if (hit >> i & 1) again[i] = 1;
  __syncthreads();
  const int kn = (a.kbytes + 15) >> 4, vn = (a.vbytes + 15) >> 4;
  const int per_row = a.heads * (kn + vn);
  for (int u = tid; u < n * per_row; u += 256) {
    const int i = u / per_row;
    int c = u - i * per_row;
    const int64_t s = place[i];
    if (s < 0 || again[i]) continue;
    const uint32_t page = (uint32_t)s / a.page, at = (uint32_t)s - page * a.page;
    const int64_t r = r0 + i;
    const char* src;
    char* dst;
    int bytes;
    if (c < a.heads * kn) {
      const int h = c / kn;
      c -= h * kn;
      src = a.k + r * a.kT + h * a.kH;
      dst = a.kc + page * a.kcP + at * a.kcS + h * a.kcH;
      bytes = a.kbytes;
    } else {
      c -= a.heads * kn;
      const int h = c / vn;
      c -= h * vn;
      src = a.v + r * a.vT + h * a.vH;
      dst = a.vc + page * a.vcP + at * a.vcS + h * a.vcH;
      bytes = a.vbytes;
    }
    const int e = 16 * c;
    if (e + 16 <= bytes) {
      *reinterpret_cast<u32x4_any_t*>(dst + e) = load_16(src + e);
    } else {
      if constexpr (E == 4) copy_tail<uint32_t>(src, dst, e, bytes);
      else copy_tail<uint16_t>(src, dst, e, bytes);
    }
  }
}

}  // namespace biops

using namespace biops;

extern "C" int biops_paged_write(int dtype, int64_t rows, int64_t heads, int64_t d, int64_t dv, const void* k,
                                 int64_t skT, int64_t skH, const void* v, int64_t svT, int64_t svH, void* kc,
                                 int64_t skcP, int64_t skcS, int64_t skcH, void* vc, int64_t svcP, int64_t svcS,
                                 int64_t svcH, int64_t pages, int64_t page_size, const void* slots, int slots64,
                                 int64_t slot_stride, int* flag, void* stream) {
  const int elt = is_float_dtype(dtype) ? dtype_bytes(dtype) : 0;
  if (elt == 0) return fail(BIOPS_ERR_DTYPE, "biops_paged_write: unsupported dtype %d", dtype);
  if (rows < 0 || heads < 0 || d < 0 || dv < 0 || pages < 0 || page_size < 0 || rows > (INT64_C(1) << 40))
    return fail(BIOPS_ERR_ARG, "biops_paged_write: negative or huge size");
  if (page_size > 0 && pages > INT64_C(0x7fffffff) / page_size)
    return fail(BIOPS_ERR_ARG, "biops_paged_write: a cache of more than 2^31 - 1 slots");
  if (heads > 0 && d + dv > (1 << 20) / heads) return fail(BIOPS_ERR_ARG, "biops_paged_write: rows of more than 2^20 elements");
  if (rows == 0 || heads == 0 || d + dv == 0) return BIOPS_OK;
  if (!slots || !flag || (d > 0 && !k) || (dv > 0 && !v)) return fail(BIOPS_ERR_ARG, "biops_paged_write: null pointer");
  if (pages * page_size > 0 && ((d > 0 && !kc) || (dv > 0 && !vc)))
    return fail(BIOPS_ERR_ARG, "biops_paged_write: null cache");
  WriteArgs a;
  a.kc = static_cast<char*>(kc), a.vc = static_cast<char*>(vc);
  a.kT = elt * skT, a.kH = elt * skH, a.vT = elt * svT, a.vH = elt * svH;
  a.kcP = elt * skcP, a.kcS = elt * skcS, a.kcH = elt * skcH;
  a.vcP = elt * svcP, a.vcS = elt * svcS, a.vcH = elt * svcH;
  a.slot_stride = slot_stride, a.flag = flag;
  a.total = (uint32_t)(pages * page_size), a.page = page_size > 0 ? (uint32_t)page_size : 1u;
  a.heads = (int)heads, a.kbytes = (int)(elt * d), a.vbytes = (int)(elt * dv);
  a.slots64 = slots64 != 0;
  for (int64_t r = 0; r < rows; r += kWriteRows) {
    a.rows = (int)(rows - r < kWriteRows ? rows - r : kWriteRows);
    a.k = static_cast<const char*>(k) + r * a.kT;
    a.v = static_cast<const char*>(v) + r * a.vT;
    a.slots = static_cast<const char*>(slots) + r * slot_stride * (slots64 ? 8 : 4);
    const dim3 grid((unsigned)cdiv(a.rows, kWriteGroup));
    if (elt == 4) hipLaunchKernelGGL((paged_write_kernel<4>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    else hipLaunchKernelGGL((paged_write_kernel<2>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    const int rc = check_launch("paged_write_kernel");
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}

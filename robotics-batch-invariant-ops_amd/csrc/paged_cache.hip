// Writes rows of new keys and values into a cache in pages.
//
// Row r goes to slot s = slots[r]: page s / page_size, place s % page_size, all heads.  A negative slot
// leaves the row out (padding); a slot past the cache is left out too and reported through the flag.
// Pure data movement: each row is read and written once, and the copy's rate is the bound.
//
// Of rows that name one slot the last stays, whatever order workgroups run in: a workgroup looks
// through the slots behind its rows and leaves a row out whose slot comes again.  It does so while its own
// rows are on their way into registers, and compares with the smallest and largest of its slots first,
// which two instructions settle where a prompt's slots lie together.  The search is quadratic, so rows go in
// launches of kWriteRows, whose order on the stream does the rest.
//
// us for rows of 8 + 8 heads of 128 fp16 (4 KB, read from memory and written): 16383 rows 29.5 (4.55 TB/s; a plain
// copy 27), with every slot somewhere else 34, and 36 / 45 with stores that stay in the caches; 48 rows of half
// that 3.2, of which a launch is 2.6.
#include "cache_slots.h"

namespace biops {

// (kWriteRows of 16384: 33.5 us for the 29.5 above)

// Rows of a workgroup: one as long as that does not fill the card, then eight, which share a search.
// us (one / eight) at 2 KB a row: 48 rows 3.2 / 5.0, 1024 4.1 / 5.3, 2048 5.7 / 5.4; 16383 rows of 4 KB 55 / 29
// (four: 38, sixteen: 35; all with cached rows and stores).
constexpr int kWriteGroup = 8, kWriteFew = 1024;

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

// E: bytes of an element; G: rows of a workgroup.
template <int E, int G>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
  __shared__ int64_t place[G];
  __shared__ int again[G];
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * G;
  const int n = a.rows - r0 < G ? a.rows - r0 : G;
  auto slot = [&](int r) -> int64_t {
    return a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[r * a.slot_stride]
                     : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[r * a.slot_stride];
  };
  int64_t first = -1;
  if (tid < n) first = slot(r0 + tid);

  // 16-byte pieces of a row: the keys of all heads, then their values.  A thread keeps one piece of every
  // `step`-th row, and another 256 pieces further on where rows are longer than that.
  const int kn = (a.kbytes + 15) >> 4, vn = (a.vbytes + 15) >> 4;
  const int per_row = a.heads * (kn + vn);
  const int step = per_row < 256 ? 256 / per_row : 1;
  const int i0 = per_row < 256 ? tid / per_row : 0;
  for (int base = 0; base < per_row; base += 256) {
    const int c = base + (per_row < 256 ? tid - i0 * per_row : tid);
    const bool active = c < per_row && i0 < step;
    const bool value = c >= a.heads * kn;
    const int x = value ? c - a.heads * kn : c;
    const int h = active ? x / (value ? vn : kn) : 0;
    const int e = 16 * (x - h * (value ? vn : kn));
    const bool whole = e + 16 <= (value ? a.vbytes : a.kbytes);
    const int64_t sT = value ? a.vT : a.kT;
    const char* const src = (value ? a.v + h * a.vH : a.k + h * a.kH) + e;
    char* const dst = (value ? a.vc + h * a.vcH : a.kc + h * a.kcH) + e;
    const int64_t dP = value ? a.vcP : a.kcP, dS = value ? a.vcS : a.kcS;
    u32x4_t piece[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int i = i0 + j * step;
      if (active && whole && i < n) piece[j] = load_16(src + (r0 + i) * sT);
    }
    if (base == 0) {  // the rows are on their way: which of them stay?
      slots_that_stay<G>(slot, r0, a.rows, first, a.total, a.flag, place, again);
    }
    if (!active) continue;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int i = i0 + j * step;
      if (i >= n) break;
      const int64_t s = place[i];
      if (s < 0 || again[i]) continue;
      const uint32_t page = (uint32_t)s / a.page, at = (uint32_t)s - page * a.page;
      char* const to = dst + page * dP + at * dS;
      if (whole) {
        // Many rows pass the caches by: they are read again a token later at the earliest.
        if constexpr (G > 1) __builtin_nontemporal_store(piece[j], reinterpret_cast<u32x4_any_t*>(to));
        else *reinterpret_cast<u32x4_any_t*>(to) = piece[j];
      } else {
        const char* from = src + (r0 + i) * sT;
        const int left = (value ? a.vbytes : a.kbytes) - e;
        if constexpr (E == 4) copy_tail<uint32_t>(from, to, 0, left);
        else copy_tail<uint16_t>(from, to, 0, left);
      }
    }
  }
}

template <int E>
static int write_launch(const WriteArgs& a, hipStream_t s) {
  const int group = a.rows <= kWriteFew ? 1 : kWriteGroup;
  const dim3 grid((unsigned)cdiv(a.rows, group));
  if (group == 1) hipLaunchKernelGGL((paged_write_kernel<E, 1>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((paged_write_kernel<E, kWriteGroup>), grid, dim3(256), 0, s, a);
  return check_launch("paged_write_kernel");
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
    const int rc = elt == 4 ? write_launch<4>(a, static_cast<hipStream_t>(stream))
                            : write_launch<2>(a, static_cast<hipStream_t>(stream));
    if (rc != BIOPS_OK) return rc;
  }
  return BIOPS_OK;
}

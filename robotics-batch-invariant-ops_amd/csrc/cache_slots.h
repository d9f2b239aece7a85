// Slots of new rows of a cache in pages: which of a workgroup's rows stay.
#pragma once

#include "biops_common.h"

namespace biops {

constexpr int kWriteRows = 8192;  // rows of a launch of a kernel that writes a cache: the search below is quadratic

// A workgroup of 256 threads with rows r0 .. r0 + G - 1 of `rows`, whose slots threads 0 .. G - 1 have in `first` (-1: none).
// place[i] becomes the slot of row r0 + i, or -1 where it names none (one past the cache sets the flag), and again[i] is set
// where a row behind it names the same slot.  The slots are compared with the smallest and largest of the workgroup's first.
template <int G, typename Slot>
__device__ __forceinline__ void slots_that_stay(Slot slot, int r0, int rows, int64_t first, uint32_t total, int* flag,
                                                int64_t* place, int* again) {
  const int tid = threadIdx.x;
  if (tid < G) {
    if (first >= (int64_t)total) {
      *flag = 1;
      first = -1;
    }
    place[tid] = first;
    again[tid] = 0;
  }
  __syncthreads();
  int64_t lo = -1, hi = -1;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int64_t s = place[i];
    if (s < 0) continue;
    lo = lo < 0 || s < lo ? s : lo;
    hi = s > hi ? s : hi;
  }
  if (hi >= 0) {
    constexpr int kAhead = 4;
    for (int r = r0 + 1; r < rows; r += 256 * kAhead) {
      int64_t s[kAhead];
      int at[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        at[j] = r + tid + 256 * j < rows ? r + tid + 256 * j : rows - 1;
        s[j] = slot(at[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (s[j] < lo || s[j] > hi) continue;
        for (int i = 0; i < G; ++i)
          if (s[j] == place[i] && at[j] > r0 + i) again[i] = 1;
      }
    }
  }
  __syncthreads();
}

}  // namespace biops

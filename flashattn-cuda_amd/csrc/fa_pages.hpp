// fa_pages.hpp — what the page writers and readers share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fa {
namespace pages {

constexpr int kPageSize = 16;
constexpr int kThreads = 256;

// Whether a token of positions [p0, p0 + n) has no valid page: checked page by
// page by the workgroup's threads.
__device__ __forceinline__ bool any_bad(const int32_t* __restrict__ pt, int64_t p0, int n,
                                        int max_pages, int num_pages) {
  if (n <= 0) return false;   // the same in every thread
  const int64_t p1 = p0 + n;
  bool bad = p0 < 0 || p1 > (int64_t)max_pages * kPageSize;
  if (!bad) {
    const int last = (int)((p1 - 1) / kPageSize);
    for (int i = (int)(p0 / kPageSize) + (int)threadIdx.x; i <= last; i += kThreads) {
      const int pid = pt[i];
      bad |= pid < 0 || pid >= num_pages;
    }
  }
  return __syncthreads_or(bad);
}

}  // namespace pages
}  // namespace fa

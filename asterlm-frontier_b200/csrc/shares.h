// Arithmetic of work cut into equal contiguous shares, in host and device code.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define ASTERQ_SHARES __host__ __device__ __forceinline__
#else
#define ASTERQ_SHARES inline
#endif

namespace asterq {

// a b / d of numbers that are not negative, b at most 1024; in 32 bits where that holds it, since a 64-bit division takes some
// hundred cycles
ASTERQ_SHARES long long share_of(long long a, int b, long long d) {
  return a < (1 << 22) && d < (1ll << 31) ? (long long)((uint32_t)a * (uint32_t)b / (uint32_t)d) : a * b / d;
}

// Share i of n is [share_of(total, i, n), share_of(total, i + 1, n)).  The number of shares from `first` on to the one that has the
// work before `end`, 0 < end <= total.
ASTERQ_SHARES int shares_up_to(long long end, int n, long long total, int first) {
  const long long last =
      end < (1 << 22) && total < (1ll << 31) ? (long long)(((uint32_t)end * (uint32_t)n - 1) / (uint32_t)total) : (end * n - 1) / total;
  return (int)last - first + 1;
}

}  // namespace asterq

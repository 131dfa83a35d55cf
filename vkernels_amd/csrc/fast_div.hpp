// fast_div.hpp — division of a non-negative int by a divisor known at the launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vk {

// n / d for 0 <= n < 2^31 as a product: with l = ceil(log2 d) and m = floor(2^(31 + l) / d) + 1,
// m d exceeds 2^(31 + l) by at most 2^l, so that floor(n m / 2^(31 + l)) = floor(n / d).
struct FastDiv {
  uint32_t magic;
  int shift;      // -1: the divisor is 1
};

inline FastDiv fast_div(int d) {
  if (d == 1) return FastDiv{0, -1};
  int l = 0;
  while ((1ll << l) < d) ++l;
  return FastDiv{(uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)d + 1), l - 1};
}

__device__ __forceinline__ int divided(int n, FastDiv f) {
  return f.shift < 0 ? n : (int)(__umulhi((uint32_t)n, f.magic) >> f.shift);
}

}  // namespace vk

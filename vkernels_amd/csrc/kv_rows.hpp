// kv_rows.hpp — device code that the kernels over new rows of a paged cache share: E4M3 codes, and the
// sequence that a row belongs to.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vk {

typedef __attribute__((ext_vector_type(4))) uint32_t kv_u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t kv_u32x2;

// What does not fit into E4M3 is stored as its largest finite code.
__device__ __forceinline__ float e4m3_range(float x) {
  // (comparisons that leave a NaN a NaN)
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}

__device__ __forceinline__ float f16_bits_to_f32(uint32_t bits, bool bf16) {
  if (bf16) return __uint_as_float(bits << 16);
  union { uint16_t u; _Float16 h; } c;
  c.u = (uint16_t)bits;
  return (float)c.h;
}

// Four values as E4M3 codes.
__device__ __forceinline__ uint32_t e4m3x4(const float* f) {
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(f[0]), e4m3_range(f[1]), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(f[2]), e4m3_range(f[3]), c, true);
}

// 8 values of a row, divided by the scale, as E4M3 codes.
__device__ __forceinline__ kv_u32x2 e4m3_codes(kv_u32x4 x, float scale, bool bf16) {
  kv_u32x2 codes;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = x[2 * i + j / 2];
      f[j] = f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xFFFFu, bf16) / scale;
    }
    codes[i] = e4m3x4(f);
  }
  return codes;
}

// The last i in [0, n) with at(i) <= x, at growing with i (0 where there is none): 64 candidates at a time,
// by the whole wavefront.
template <class F>
__device__ __forceinline__ int last_not_above(int n, int x, F at) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const uint64_t below = __ballot(i < hi && at(i) <= x);
    const int found = max(1, (int)__popcll(below));
    hi = min(hi, lo + found * step);
    lo += (found - 1) * step;
  }
  return lo;
}

}  // namespace vk

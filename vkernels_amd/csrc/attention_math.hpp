// attention_math.hpp — device code that the attention kernels share: types of the matrix instructions, E4M3 codes
// as 16-bit values, exponentials, capped scores.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vk {
namespace attention {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();
// The reference of the exponentials is moved when the scores pass it by more than 2^8: weights of
// up to 256 cost no accuracy, and few tiles then have to rescale what they have summed.
constexpr float kSlack = 8.0f;

// The 16-bit type that the matrix instructions multiply in.
struct Bf16 {
  static constexpr bool kTileScale = false;
  typedef __bf16 T;
  typedef __attribute__((ext_vector_type(8))) __bf16 V8;
  typedef __attribute__((ext_vector_type(2))) __bf16 V2;
  static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ V2 of_fp8(uint32_t codes, bool high) {
    return high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true)
                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false);
  }
};
struct F16 {
  static constexpr bool kTileScale = true;
  typedef _Float16 T;
  typedef __attribute__((ext_vector_type(8))) _Float16 V8;
  typedef __attribute__((ext_vector_type(2))) _Float16 V2;
  static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ V2 of_fp8(uint32_t codes, bool high) {
    return high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true)
                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false);
  }
};

template <class M>
__device__ __forceinline__ typename M::V8 as_v8(u32x4 x) {
  union { u32x4 u; typename M::V8 v; } c;
  c.u = x;
  return c.v;
}

// 8 E4M3 codes -> 8 values (exact in either type).
template <class M>
__device__ __forceinline__ typename M::V8 fp8x8(uint32_t lo, uint32_t hi) {
  union { typename M::V2 p[4]; typename M::V8 v; } c;
  c.p[0] = M::of_fp8(lo, false);
  c.p[1] = M::of_fp8(lo, true);
  c.p[2] = M::of_fp8(hi, false);
  c.p[3] = M::of_fp8(hi, true);
  return c.v;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// log of a row's sum ll 2^ref (a sink alone is handed back as it is).
__device__ __forceinline__ float log_of_sum(float ref, float ll, const float* sink) {
  if (ll == 0.0f) return kNegInf;
  if (sink != nullptr && ll == 1.0f && ref == *sink * kLog2e) return *sink;
  return ref * kLn2 + logf(ll);
}
__device__ __forceinline__ float or_zero(float m) { return m == kNegInf ? 0.0f : m; }

// A score capped, in powers of two: z2 is twice the score over the cap, cap_out the cap.
// c tanh(y / c) = c (1 - 2 / (1 + e^{2 y / c})), and y (1 - z^2 / 3 + 2 z^4 / 15) with z = y / c below 0.1, where
// the first form cancels.  Hardware exponential and reciprocal leave less than 2^-20 of the cap.
__device__ __forceinline__ float capped(float z2, float cap_out) {
  const float big = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + exp2_fast(z2));
  const float z = z2 * (0.5f * kLn2), zz = z * z;
  const float small = z * (1.0f - zz * (0.33333334f - zz * 0.13333334f));
  return cap_out * (fabsf(z) < 0.1f ? small : big);
}

// An array of int32 that the kernel only reads: through the scalar cache where the index is uniform.
typedef const __attribute__((address_space(4))) int32_t* ConstInts;
__device__ __forceinline__ ConstInts read_only(const int32_t* p) { return (ConstInts)(uintptr_t)p; }

}  // namespace attention
}  // namespace vk

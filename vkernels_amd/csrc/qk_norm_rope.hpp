// qk_norm_rope.hpp — launcher of the norm and rotation of queries and keys (qk_norm_rope.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fast_div.hpp"

namespace vk {

constexpr int kRopeAxes = 4;

struct QkNormRopeArgs {
  const void* q;            // [T, Hq, D], rows of D values 16-byte aligned
  const void* k;            // [T, Hkv, D]
  void* q_out;
  void* k_out;
  const void* q_weight;     // [D] or null
  const void* k_weight;
  const int32_t* positions; // [axes, T]
  const float* inv_freq;    // [turned / 2]
  int64_t q_stride_t, q_stride_h, k_stride_t, k_stride_h;           // elements
  int64_t qo_stride_t, qo_stride_h, ko_stride_t, ko_stride_h;
  int64_t axis_stride;
  int T, Hq, Hkv, D, turned;
  int section_end[kRopeAxes];   // frequencies of axes 0 .. i; the last one used is turned / 2
  int axes;
  float eps, factor;
  bool norm, weights_f32;
  // (set by the launcher)
  int lanes;                // of a row: a power of two
  int rows;                 // of a wavefront at a time
  int per_wave;             // times that many
  int waves;                // of a token
  FastDiv by_waves;
  float inv_width;
};
void launch_qk_norm_rope(const QkNormRopeArgs& a, bool bf16, bool pairs, hipStream_t stream);

}  // namespace vk

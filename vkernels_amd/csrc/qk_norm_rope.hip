// qk_norm_rope.hip — RMS norm of every query and key head and the rotation by the token's position.
//
// A row x of D values becomes y = x w / sqrt(mean x^2 + eps); its first 2 R values are R pairs, the i-th
// turned by the angle p f_i, where p is the token's position on the axis that frequency i belongs to:
//   (a, b) -> factor (a cos - b sin, b cos + a sin).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "qk_norm_rope.hpp"

namespace vk {
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int kWaves = 4;           // of a workgroup
constexpr int kMostFreqs = 128;     // half a row

// V 16-bit values that a lane loads at once: 16 or 8 bytes.
template <int V>
using Piece = __attribute__((ext_vector_type(V / 2))) uint32_t;

template <bool BF16>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  if constexpr (BF16) return __uint_as_float(bits << 16);
  union { uint16_t u; _Float16 h; } c;
  c.u = (uint16_t)bits;
  return (float)c.h;
}
template <bool BF16>
__device__ __forceinline__ uint32_t to_bits(float x) {
  if constexpr (BF16) {
    union { __bf16 b; uint16_t u; } c;
    c.b = (__bf16)x;
    return c.u;
  }
  union { _Float16 h; uint16_t u; } c;
  c.h = (_Float16)x;
  return c.u;
}

template <int V, bool BF16>
__device__ __forceinline__ void widen(const Piece<V>& p, float* x) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    x[2 * i] = to_f32<BF16>(p[i] & 0xFFFFu);
    x[2 * i + 1] = to_f32<BF16>(p[i] >> 16);
  }
}
template <int V, bool BF16>
__device__ __forceinline__ Piece<V> narrow(const float* x) {
  Piece<V> p;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) p[i] = to_bits<BF16>(x[2 * i]) | to_bits<BF16>(x[2 * i + 1]) << 16;
  return p;
}

// A wavefront takes heads of one token, a.rows at a time.  A lane has two pieces of V values of a row: those
// whose values are each other's partners (V values at i and the V at i + R; of neighbouring pairs any two), so that a
// pair never leaves its lane, and it has the same pieces of every row, so that its V cosines and sines are loaded
// once.  The angles of a token are worked out once a wavefront, a lane for each
// frequency: the product in 64 bits, of which the whole turns go before it is cut to 32 (a position of 2^20
// leaves 32 bits no more than an eighth of a radian at a frequency of 1).
// Bound by the rows read and written.  PAST: results of more bytes than the L2 caches hold go past them (8191 tokens,
// 40 heads of 128, 168 MB: 43 us with stores through the caches, 35 past them).
template <int V, bool BF16, bool PAIRS, bool PAST>
__global__ __launch_bounds__(64 * kWaves) void qk_norm_rope_kernel(const QkNormRopeArgs a) {
  __shared__ __attribute__((aligned(16))) float cos_lds[kWaves][kMostFreqs], sin_lds[kWaves][kMostFreqs];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = (int64_t)blockIdx.x * kWaves + wave;
  if (at >= (int64_t)a.T * a.waves) return;
  const int t = divided((int)at, a.by_waves), part = (int)at - t * a.waves;
  const int freqs = a.turned / 2, heads = a.Hq + a.Hkv;
  const int unit = lane & (a.lanes - 1), sub = lane / a.lanes;
  const bool in_row = unit * 2 * V < a.D;
  // where the lane's two pieces lie (lanes without any read the first ones), and whether they turn
  const bool beside = !PAIRS && unit * V >= freqs;
  const int at0 = !in_row ? 0 : beside ? unit * 2 * V : unit * V;
  const int at1 = !in_row ? V : PAIRS ? at0 + a.D / 2 : beside ? at0 + V : at0 + freqs;
  const bool turns0 = PAIRS ? at0 < a.turned : !beside, turns1 = PAIRS ? at1 < a.turned : !beside;

  const int head0 = part * a.per_wave * a.rows;
  const int last = min(heads, head0 + a.per_wave * a.rows) - 1;
  auto row_of = [&](int h, const char* q, const char* k, int64_t qt, int64_t qh, int64_t kt, int64_t kh) {
    return h < a.Hq ? q + (t * qt + h * qh) * 2 : k + (t * kt + (h - a.Hq) * kh) * 2;
  };
  auto load = [&](int h, Piece<V>& x, Piece<V>& y) {
    const char* const row = row_of(min(h, last), (const char*)a.q, (const char*)a.k, a.q_stride_t, a.q_stride_h,
                                   a.k_stride_t, a.k_stride_h);
    x = *(const Piece<V>*)(row + at0 * 2);
    y = *(const Piece<V>*)(row + at1 * 2);
  };
  Piece<V> x, y;
  load(head0 + sub, x, y);

  __attribute__((aligned(16))) float wq[2 * V], wk[2 * V];
  auto load_weights = [&](const void* w, float* to) {
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) to[i] = 1.0f;
    if (w == nullptr) return;
    if (a.weights_f32) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        *(f32x4*)(to + i) = *(const f32x4*)((const float*)w + at0 + i);
        *(f32x4*)(to + V + i) = *(const f32x4*)((const float*)w + at1 + i);
      }
    } else {
      widen<V, BF16>(*(const Piece<V>*)((const char*)w + at0 * 2), to);
      widen<V, BF16>(*(const Piece<V>*)((const char*)w + at1 * 2), to + V);
    }
  };
  load_weights(a.q_weight, wq);
  load_weights(a.k_weight, wk);

  for (int i = lane; i < freqs; i += 64) {
    int axis = 0;
#pragma unroll
    for (int j = 0; j + 1 < kRopeAxes; ++j)
      if (j + 1 < a.axes && i >= a.section_end[j]) axis = j + 1;
    const int p = a.positions[axis * a.axis_stride + t];
    const double turns_of = (double)p * (double)a.inv_freq[i] * 0.15915494309189533577;   // 1 / 2 pi
    float s, c;
    sincospif(2.0f * (float)(turns_of - rint(turns_of)), &s, &c);
    cos_lds[wave][i] = c * a.factor;
    sin_lds[wave][i] = s * a.factor;
  }
  // (lanes read what other lanes of their wavefront wrote: LDS keeps the order, and so must the compiler)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  float co[V], si[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = !PAIRS ? unit * V + i : i < V / 2 ? at0 / 2 + i : at1 / 2 + i - V / 2;
    const bool turns = PAIRS && i >= V / 2 ? turns1 : turns0;
    co[i] = turns ? cos_lds[wave][at] : 1.0f;
    si[i] = turns ? sin_lds[wave][at] : 0.0f;
  }

  for (int i = 0; i < a.per_wave; ++i) {
    const int h = head0 + i * a.rows + sub;
    if (head0 + i * a.rows > last) break;
    float v[2 * V];
    widen<V, BF16>(x, v);
    widen<V, BF16>(y, v + V);
    if (i + 1 < a.per_wave) load(h + a.rows, x, y);
    if (a.norm) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) sum += v[j] * v[j];
      if (!in_row) sum = 0.0f;
      for (int d = 1; d < a.lanes; d <<= 1) sum += __shfl_xor(sum, d);
      const float inv = rsqrtf(sum * a.inv_width + a.eps);
      const bool query = h < a.Hq;
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) v[j] = v[j] * inv * (query ? wq[j] : wk[j]);
    }
    float o[2 * V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      // (of halves a piece each, of neighbours both in one; values beside the pairs have cosine 1 and sine 0,
      // and a product with that 0 is none where the partner is infinite)
      const int p0 = PAIRS ? 2 * j : j, p1 = PAIRS ? 2 * j + 1 : V + j;
      const bool turns = PAIRS && j >= V / 2 ? turns1 : turns0;
      o[p0] = turns ? v[p0] * co[j] - v[p1] * si[j] : v[p0];
      o[p1] = turns ? v[p1] * co[j] + v[p0] * si[j] : v[p1];
    }
    if (in_row && h <= last) {
      char* const row = (char*)row_of(h, (const char*)a.q_out, (const char*)a.k_out, a.qo_stride_t, a.qo_stride_h,
                                      a.ko_stride_t, a.ko_stride_h);
      if constexpr (PAST) {
        __builtin_nontemporal_store(narrow<V, BF16>(o), (Piece<V>*)(row + at0 * 2));
        __builtin_nontemporal_store(narrow<V, BF16>(o + V), (Piece<V>*)(row + at1 * 2));
      } else {
        *(Piece<V>*)(row + at0 * 2) = narrow<V, BF16>(o);
        *(Piece<V>*)(row + at1 * 2) = narrow<V, BF16>(o + V);
      }
    }
  }
}

template <int V, bool BF16, bool PAIRS>
void launch_pieces(const QkNormRopeArgs& a, hipStream_t stream) {
  const dim3 grid((uint32_t)(((int64_t)a.T * a.waves + kWaves - 1) / kWaves)), block(64 * kWaves);
  // (rows of 128 bytes and less, and pieces that lie side by side, would go past the caches as parts of lines: 64 values
  // 30 us through them and 33 past, pairs in pieces side by side 36 and 39)
  const bool past = (int64_t)a.T * (a.Hq + a.Hkv) * a.D * 2 > 32 << 20 && a.D >= 128 && (PAIRS || a.turned == a.D);
  if constexpr (V == 8) {
    if (past) {
      hipLaunchKernelGGL((qk_norm_rope_kernel<V, BF16, PAIRS, true>), grid, block, 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((qk_norm_rope_kernel<V, BF16, PAIRS, false>), grid, block, 0, stream, a);
}

template <bool BF16>
void launch_type(const QkNormRopeArgs& a, bool pairs, int V, hipStream_t stream) {
  if (pairs)
    launch_pieces<8, BF16, true>(a, stream);
  else if (V == 8)
    launch_pieces<8, BF16, false>(a, stream);
  else
    launch_pieces<4, BF16, false>(a, stream);
}

}  // namespace

void launch_qk_norm_rope(const QkNormRopeArgs& args, bool bf16, bool pairs, hipStream_t stream) {
  QkNormRopeArgs a = args;
  // pieces of 8 values, or of 4 where the partners of 8 would not start on a piece
  const int V = pairs || a.turned % 16 == 0 ? 8 : 4;
  const int units = a.D / (2 * V);
  a.lanes = 1;
  while (a.lanes < units) a.lanes *= 2;
  a.rows = 64 / a.lanes;
  // A wavefront for all heads of a token, so that its angles are worked out once; where tokens are few, for
  // fewer heads, down to those that it takes at once.
  const int times = (a.Hq + a.Hkv + a.rows - 1) / a.rows;
  const int split = std::min(times, std::max(1, 4096 / a.T));
  a.per_wave = (times + split - 1) / split;
  a.waves = (times + a.per_wave - 1) / a.per_wave;
  a.by_waves = fast_div(a.waves);
  a.inv_width = 1.0f / (float)a.D;
  if (bf16) launch_type<true>(a, pairs, V, stream); else launch_type<false>(a, pairs, V, stream);
}

}  // namespace vk

// kv_blocks.hip — a paged key-value cache of E4M3 codes with a scale for each block of positions and head:
// new rows quantised as they are written, and positions read back as ordinary rows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "kv_blocks.hpp"
#include "kv_rows.hpp"

namespace vk {
namespace {

typedef kv_u32x4 u32x4;
typedef kv_u32x2 u32x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;

constexpr int kRowLoads = 4;     // pieces of new rows that a lane holds
constexpr int kOldLoads = 4;     // pieces of older codes that it asks for at once

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;

// The largest magnitudes of the lower and of the upper halves' 16-bit values, as their bits (which order as they do).
__device__ __forceinline__ uint32_t larger_halves(uint32_t x, uint32_t y) {
  union { uint32_t u; u16x2 v; } a, b;
  a.u = x & 0x7FFF7FFFu;
  b.u = y & 0x7FFF7FFFu;
  a.v = __builtin_elementwise_max(a.v, b.v);
  return a.u;
}
// ... with zeros for what is no finite number (an exponent of ones carries into the half's sign).
__device__ __forceinline__ uint32_t finite_halves(uint32_t x, bool bf16) {
  const uint32_t bad = ((x & (bf16 ? 0x7F807F80u : 0x7C007C00u)) + (bf16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
  return x & ~((bad >> 15) * 0xFFFFu);
}
__device__ __forceinline__ uint32_t largest_halves(uint32_t size, u32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) size = larger_halves(size, x[i]);
  return size;
}
__device__ __forceinline__ u32x4 finite_values(u32x4 x, bool bf16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = finite_halves(x[i], bf16);
  return x;
}
__device__ __forceinline__ uint32_t larger_half(uint32_t size) { return max(size & 0xFFFFu, size >> 16); }
__device__ __forceinline__ uint32_t infinity_of(bool bf16) { return bf16 ? 0x7F80u : 0x7C00u; }

// Division by a block's scale.  With r the reciprocal, correctly rounded, and q = x r rounded, q + (x - q s) r is the
// quotient of an x that is not 0, correctly rounded, unless the scale's significand is all ones (Markstein 1990) or the
// remainder leaves the range of 32-bit floats: such scales are divided by.  (A code's rounding looks at quotients from
// 2^-11 on, so that scales from 2^-80 to 2^80 keep all of it in range.)
constexpr int kZeroOrNoNumber = 0x267;      // of v_cmp_class: zeros, infinities and NaN of either sign
struct Scale {
  float s, r;
  bool simple;
  __device__ __forceinline__ explicit Scale(float scale) {
    // (a block of zeros has scale 0, and its codes are zeros)
    s = scale > 0.0f ? scale : 1.0f;
    r = 1.0f / s;
    simple = s >= 0x1p-80f && s <= 0x1p80f && (__float_as_uint(s) & 0x7FFFFFu) != 0x7FFFFFu;
  }
  __device__ __forceinline__ float divided(float x) const {
    const float q = x * r;
    return __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  }
};
__device__ __forceinline__ u32x2 codes_by(u32x4 x, const Scale& by, bool bf16) {
  if (!by.simple) return e4m3_codes(x, by.s, bf16);
  u32x2 codes;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = x[2 * i + j / 2];
      const float v = f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xFFFFu, bf16), q = by.divided(v);
      f[j] = __builtin_amdgcn_classf(v, kZeroOrNoNumber) ? v : q;      // (as they are: of -0 the remainder loses the sign)
    }
    codes[i] = e4m3x4(f);
  }
  return codes;
}

// 8 codes times a factor, as codes.
__device__ __forceinline__ u32x2 scaled_codes(u32x2 c, float factor) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], true);
    const float f[4] = {p[0] * factor, p[1] * factor, q[0] * factor, q[1] * factor};
    c[w] = e4m3x4(f);
  }
  return c;
}

// A block of positions has one scale for a head: s = max(s of its older positions, max |x| / 448 over its new
// rows), codes the E4M3 values nearest to x / s.  Where s grows, the older codes c become those nearest to
// c (s_old / s).
// A wavefront, or of larger blocks a workgroup, takes the keys or the values of one block in one head: nobody else
// touches them, so that the codes can be read, scaled and written back without an order among them.  Its lanes hold the
// new rows' pieces of 8 values (up to 4 each; of still larger blocks they are read again for the second pass, from the
// cache).  Bound by a chain of dependent loads (the sequence, its length, its page, the block's scale) beside the rows',
// and by the vector instructions of the codes: 8191 tokens of 8 heads of 128 in blocks of 16, 50 MB, in 14.4 us (18 with
// IEEE divisions; keys and values by one wavefront 23), in blocks of 64 17 (43 by wavefronts); 255 single tokens 5.6.
template <bool RAGGED, bool WORKGROUP>
__global__ __launch_bounds__(256) void kv_quantise_kernel(const KvQuantiseArgs A, int bf16_) {
  constexpr int kLanes = WORKGROUP ? 256 : 64;
  __shared__ uint32_t size_lds[4];
  const KvAppendArgs& a = A.a;
  const bool bf16 = bf16_ != 0;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = WORKGROUP ? threadIdx.x : threadIdx.x & 63;
  const int64_t at = WORKGROUP ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (at >= (int64_t)A.slots * a.Hkv * 2) return;
  const int unit = (int)(at >> 1), is_v = (int)(at & 1);
  const int slot = divided(unit, A.by_heads), h = unit - slot * a.Hkv;

  int b = slot, k = 0, s0 = slot, s1 = slot + 1;
  if constexpr (RAGGED) {
    auto base = [&](int i) { return divided(min(max(a.starts[i], 0), a.tokens), A.by_block) + 2 * i; };
    b = last_not_above(a.B, slot, base);
    k = slot - base(b);
    s0 = min(max(a.starts[b], 0), a.tokens);
    s1 = min(max(a.starts[b + 1], s0), a.tokens);
    if (k < 0 || s1 == s0) return;
  }
  // New positions [lo, hi) of the sequence are rows of the tokens at them less `off`; this block's are [from, to).
  const int len = a.lens[b];
  if (len <= 0) return;
  const int off = len - s1, lo = max(0, s0 + off), hi = len;
  const int64_t begin64 = ((int64_t)divided(lo, A.by_block) + k) * A.block;
  if (begin64 >= hi) return;
  const int begin = (int)begin64, from = max(begin, lo), to = min((int64_t)begin + A.block, (int64_t)hi);
  const int in_table = divided(begin, a.by_page);
  if (in_table >= a.table_width) return;
  const int page = a.table[(int64_t)b * a.table_stride + in_table];

  const char* const rows = (const char*)(is_v ? a.v : a.k);
  const int64_t by_t = is_v ? a.v_stride_t : a.k_stride_t, by_h = is_v ? a.v_stride_h : a.k_stride_h;
  const int pieces = a.pieces, n = (to - from) * pieces;
  auto load = [&](int i) -> u32x4 {
    const int row = divided(i, a.by_pieces);
    return *(const u32x4*)(rows + ((int64_t)(from - off + row) * by_t + h * by_h + (i - row * pieces) * 8) * 2);
  };
  u32x4 x[kRowLoads];
#pragma unroll
  for (int i = 0; i < kRowLoads; ++i) x[i] = load(min(lane + kLanes * i, n - 1));
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int first_slot = begin - in_table * a.page_size;      // of the page
  float* const scale_at = (is_v ? A.v_scale : A.k_scale) + ((int64_t)page * a.Hkv + h) * A.blocks + divided(first_slot, A.by_block);
  const bool older = from > begin;
  const float before = older ? *scale_at : 0.0f;

  // (the largest magnitude, and once more without what is no finite number where there is such a value)
  auto largest = [&](bool finite) {
    uint32_t size = 0;
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) size = largest_halves(size, finite ? finite_values(x[i], bf16) : x[i]);
    for (int i = lane + kLanes * kRowLoads; i < n; i += kLanes) {
      const u32x4 y = load(i);
      size = largest_halves(size, finite ? finite_values(y, bf16) : y);
    }
    size = larger_half(size);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) size = max(size, (uint32_t)__shfl_xor((int)size, d));
    if constexpr (WORKGROUP) {
      __syncthreads();      // (twice in a row: the first sizes have been read)
      if ((threadIdx.x & 63) == 0) size_lds[wave] = size;
      __syncthreads();
      size = max(max(size_lds[0], size_lds[1]), max(size_lds[2], size_lds[3]));
    }
    return size;
  };
  uint32_t size = largest(false);
  if (size >= infinity_of(bf16)) size = largest(true);
  const float needed = f16_bits_to_f32(size, bf16) / 448.0f;
  const bool grows = older && !(before >= needed);
  const float scale = older && !grows ? before : needed;

  char* const codes = (char*)(is_v ? a.v_cache : a.k_cache) + (int64_t)page * a.page_stride + (int64_t)h * a.head_stride;
  auto code_at = [&](int position, int piece) -> u32x2* {
    return (u32x2*)(codes + (int64_t)(position - in_table * a.page_size) * a.slot_stride + piece * 8);
  };
  if (grows) {
    const float factor = before / scale;
    const int n_old = (from - begin) * pieces;
    for (int i0 = lane; i0 < n_old; i0 += kLanes * kOldLoads) {
      u32x2 c[kOldLoads];
#pragma unroll
      for (int j = 0; j < kOldLoads; ++j) {
        const int i = min(i0 + kLanes * j, n_old - 1), row = divided(i, a.by_pieces);
        c[j] = *code_at(begin + row, i - row * pieces);
      }
#pragma unroll
      for (int j = 0; j < kOldLoads; ++j) {
        const int i = i0 + kLanes * j, row = divided(i, a.by_pieces);
        if (i >= n_old) break;
        *code_at(begin + row, i - row * pieces) = scaled_codes(c[j], factor);
      }
    }
  }
  const Scale by(scale);
#pragma unroll
  for (int i = 0; i < kRowLoads; ++i) {
    const int j = lane + kLanes * i, row = divided(j, a.by_pieces);
    if (j < n) *code_at(from + row, j - row * pieces) = codes_by(x[i], by, bf16);
  }
  for (int j = lane + kLanes * kRowLoads; j < n; j += kLanes) {
    const int row = divided(j, a.by_pieces);
    *code_at(from + row, j - row * pieces) = codes_by(load(j), by, bf16);
  }
  if (lane == 0 && (grows || !older)) *scale_at = scale;
}

// Blocks of one position: a scale for each row, that nothing else touches.  A row's lanes (a power of two) take 8 values
// each of its key and its value; rows one behind the other as the append's.  8191 tokens of 8 heads of 128 take
// 18.8 us with the call (by wavefronts for a block, as above, 108).
__global__ __launch_bounds__(256) void kv_quantise_rows_kernel(const KvQuantiseArgs A, int bf16, int lanes, int lane_shift) {
  const KvAppendArgs& a = A.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t first = idx - (threadIdx.x & 63);
  if (first >= ((int64_t)a.tokens * a.Hkv << lane_shift)) return;
  const int unit = (int)min(idx >> lane_shift, (int64_t)a.tokens * a.Hkv - 1), piece = threadIdx.x & (lanes - 1);
  const bool real = idx >> lane_shift <= unit && piece < a.pieces;
  const int t = divided(unit, A.by_heads), h = unit - t * a.Hkv, d = min(piece, a.pieces - 1) * 8;
  const u32x4 k = *(const u32x4*)((const char*)a.k + ((int64_t)t * a.k_stride_t + (int64_t)h * a.k_stride_h + d) * 2);
  const u32x4 v = *(const u32x4*)((const char*)a.v + ((int64_t)t * a.v_stride_t + (int64_t)h * a.v_stride_h + d) * 2);
  uint32_t k_size = larger_half(largest_halves(0, finite_values(k, bf16 != 0)));
  uint32_t v_size = larger_half(largest_halves(0, finite_values(v, bf16 != 0)));
  for (int i = 1; i < lanes; i <<= 1) {
    k_size = max(k_size, (uint32_t)__shfl_xor((int)k_size, i));
    v_size = max(v_size, (uint32_t)__shfl_xor((int)v_size, i));
  }
  const float ks = f16_bits_to_f32(k_size, bf16 != 0) / 448.0f, vs = f16_bits_to_f32(v_size, bf16 != 0) / 448.0f;
  int seq = t;
  if (a.starts != nullptr) {
    seq = last_not_above(a.B, divided((int)(first >> lane_shift), A.by_heads), [&](int i) { return a.starts[i]; });
    while (seq + 1 < a.B && a.starts[seq + 1] <= t) ++seq;
    if (t < a.starts[seq]) return;
  }
  const int len = a.lens[seq];
  const int pos = a.starts != nullptr ? len - a.starts[seq + 1] + t : len - 1;
  if (!real || pos < 0 || pos >= len) return;
  const int in_table = divided(pos, a.by_page);
  if (in_table >= a.table_width) return;
  const int page = a.table[(int64_t)seq * a.table_stride + in_table];
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int slot = pos - in_table * a.page_size;
  const int64_t to = (int64_t)page * a.page_stride + (int64_t)h * a.head_stride + (int64_t)slot * a.slot_stride + d;
  *(u32x2*)((char*)a.k_cache + to) = codes_by(k, Scale(ks), bf16 != 0);
  *(u32x2*)((char*)a.v_cache + to) = codes_by(v, Scale(vs), bf16 != 0);
  if (piece == 0) {
    const int64_t at = ((int64_t)page * a.Hkv + h) * A.blocks + slot;
    A.k_scale[at] = ks;
    A.v_scale[at] = vs;
  }
}

// ---- reading back ----------------------------------------------------------------------------------

// 8 values of a row that is read, as they are or codes as values of 16 bits.
template <bool BF16>
__device__ __forceinline__ u32x4 row_values(u32x4 x, float) { return x; }
template <bool BF16>
__device__ __forceinline__ u32x4 row_values(u32x2 codes, float scale) {
  auto pack = [](float x, float y) -> uint32_t {
    if constexpr (BF16) {
      union { __bf16 e[2]; uint32_t u; } c;
      c.e[0] = (__bf16)x;
      c.e[1] = (__bf16)y;
      return c.u;
    } else {
      union { _Float16 e[2]; uint32_t u; } c;
      c.e[0] = (_Float16)x;
      c.e[1] = (_Float16)y;
      return c.u;
    }
  };
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[i], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[i], true);
    y[2 * i] = pack(p[0] * scale, p[1] * scale);
    y[2 * i + 1] = pack(q[0] * scale, q[1] * scale);
  }
  return y;
}

// A workgroup takes `chunk` rows in all heads: a lane each looks up where they lie, then every thread reads 8 values
// of a key and of a value in a head, four of each at a time.  Bound by the rows read and written: 60001 positions of 8
// heads of 128 in 8 bits, 369 MB, in 77 us, 4.8 TB/s.  (A thread for 8 values with look-ups of its own took 116;
// 16 codes a thread 86, stores past the caches no less than 77.)
template <bool FP8, bool BF16>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvReadArgs a) {
  typedef std::conditional_t<FP8, u32x2, u32x4> Piece;
  constexpr int kAtOnce = 4;
  __shared__ int64_t row_lds[kKvReadChunk], scale_lds[kKvReadChunk];     // (elements; -1: zeros, -2: left as it is)
  const int tid = threadIdx.x, t0 = blockIdx.x * a.chunk;
  const int rows = min(a.chunk, a.tokens - t0);
  if (tid < 64) {
    int seq = 0;
    if (a.starts != nullptr) seq = last_not_above(a.B, t0, [&](int i) { return a.starts[i]; });
    if (tid < rows) {
      const int t = t0 + tid;
      bool mine = true;          // the row belongs to a sequence
      if (a.starts != nullptr) {
        while (seq + 1 < a.B && a.starts[seq + 1] <= t) ++seq;
        mine = t >= a.starts[seq] && t < a.starts[seq + 1];
      } else {
        seq = t;
      }
      int64_t row = mine || a.clear_rest ? -1 : -2, scale = 0;
      const int len = a.lens[seq];
      const int pos = a.starts != nullptr ? len - a.starts[seq + 1] + t : len - 1;
      if (mine && pos >= 0 && pos < len) {
        const int in_table = divided(pos, a.by_page);
        const int page = in_table < a.table_width ? a.table[(int64_t)seq * a.table_stride + in_table] : -1;
        if ((uint32_t)page < (uint32_t)a.num_pages) {
          const int slot = pos - in_table * a.page_size;
          row = (int64_t)page * a.page_stride + (int64_t)slot * a.slot_stride;
          if (FP8 && a.blocks > 0) scale = (int64_t)page * a.Hkv * a.blocks + divided(slot, a.by_block);
        }
      }
      row_lds[tid] = row;
      scale_lds[tid] = scale;
    }
  }
  __syncthreads();
  constexpr int kElem = FP8 ? 1 : 2;
  const int per_row = a.Hkv * a.pieces, n = rows * per_row;
  for (int i0 = tid; i0 < n; i0 += 256 * kAtOnce) {
    Piece k[kAtOnce], v[kAtOnce];
    float ks[kAtOnce], vs[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + 256 * j;
      k[j] = v[j] = Piece{};
      ks[j] = vs[j] = 1.0f;
      if (i < n) {
        const int r = divided(i, a.by_token), rest = i - r * per_row, h = divided(rest, a.by_pieces);
        const int64_t row = row_lds[r];
        if (row >= 0) {
          const int64_t from = (row + (int64_t)h * a.head_stride + (rest - h * a.pieces) * 8) * kElem;
          k[j] = *(const Piece*)((const char*)a.k_cache + from);
          v[j] = *(const Piece*)((const char*)a.v_cache + from);
          if constexpr (FP8) {
            const int64_t s = a.blocks > 0 ? scale_lds[r] + (int64_t)h * a.blocks : h;
            ks[j] = a.k_scale[s];
            vs[j] = a.v_scale[s];
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + 256 * j;
      if (i >= n) break;
      const int r = divided(i, a.by_token), rest = i - r * per_row, h = divided(rest, a.by_pieces);
      const int d = (rest - h * a.pieces) * 8;
      if (row_lds[r] == -2) continue;
      u32x4* const k_to = (u32x4*)((char*)a.k + ((int64_t)(t0 + r) * a.k_stride_t + (int64_t)h * a.k_stride_h + d) * 2);
      u32x4* const v_to = (u32x4*)((char*)a.v + ((int64_t)(t0 + r) * a.v_stride_t + (int64_t)h * a.v_stride_h + d) * 2);
      const u32x4 k_row = row_values<BF16>(k[j], ks[j]), v_row = row_values<BF16>(v[j], vs[j]);
      *k_to = k_row;
      *v_to = v_row;
    }
  }
}

}  // namespace

void launch_kv_quantise(const KvQuantiseArgs& args, bool bf16, hipStream_t stream) {
  KvQuantiseArgs A = args;
  A.a.pieces = A.a.D / 8;
  A.a.by_page = fast_div(A.a.page_size);
  A.a.by_pieces = fast_div(A.a.pieces);
  A.by_block = fast_div(A.block);
  A.by_heads = fast_div(A.a.Hkv);
  if (A.block == 1) {
    int lanes = 1, shift = 0;
    while (lanes < A.a.pieces) lanes *= 2, ++shift;
    const int64_t threads = (int64_t)A.a.tokens * A.a.Hkv * lanes;
    hipLaunchKernelGGL(kv_quantise_rows_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, A, (int)bf16, lanes,
                       shift);
    return;
  }
  A.slots = (int)kv_quantise_slots(A.a.B, A.a.tokens, A.block, A.a.starts != nullptr);
  const int64_t units = (int64_t)A.slots * A.a.Hkv * 2;
  const bool ragged = A.a.starts != nullptr, workgroup = ragged && A.block * A.a.pieces > 64 * kRowLoads;
  const dim3 grid((unsigned)(workgroup ? units : (units + 3) / 4)), block(256);
  if (workgroup)
    hipLaunchKernelGGL((kv_quantise_kernel<true, true>), grid, block, 0, stream, A, (int)bf16);
  else if (ragged)
    hipLaunchKernelGGL((kv_quantise_kernel<true, false>), grid, block, 0, stream, A, (int)bf16);
  else
    hipLaunchKernelGGL((kv_quantise_kernel<false, false>), grid, block, 0, stream, A, (int)bf16);
}

void launch_kv_read(const KvReadArgs& args, int kind, hipStream_t stream) {
  KvReadArgs a = args;
  const bool fp8 = kind >= 2, b16 = kind % 2 == 0;
  a.pieces = a.D / 8;
  const int per_row = a.Hkv * a.pieces;
  a.by_page = fast_div(a.page_size);
  a.by_pieces = fast_div(a.pieces);
  a.by_token = fast_div(per_row);
  a.by_block = fast_div(a.blocks > 0 ? a.block : 1);
  // Work for every thread, and where there are rows enough for 2048 workgroups four times that and more.
  const int least = std::max(1, 256 / per_row), most = std::max(1, std::min(kKvReadChunk, 8192 / per_row));
  a.chunk = std::max(std::min(least, kKvReadChunk), std::min(most, a.tokens / 2048));
  const dim3 grid((unsigned)((a.tokens + a.chunk - 1) / a.chunk)), block(256);
  if (!fp8)
    hipLaunchKernelGGL((kv_read_kernel<false, true>), grid, block, 0, stream, a);
  else if (b16)
    hipLaunchKernelGGL((kv_read_kernel<true, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((kv_read_kernel<true, false>), grid, block, 0, stream, a);
}

}  // namespace vk

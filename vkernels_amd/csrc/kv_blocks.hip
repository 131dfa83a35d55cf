// kv_blocks.hip — a paged key-value cache of E4M3 codes with a scale for each block of positions and head:
// new rows quantised as they are written, and positions read back as ordinary rows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_blocks.hpp"
#include "kv_rows.hpp"

namespace vk {
namespace {

typedef kv_u32x4 u32x4;
typedef kv_u32x2 u32x2;

constexpr int kRowLoads = 4;     // pieces of new rows that a lane holds
constexpr int kOldLoads = 4;     // pieces of older codes that it asks for at once

// The largest magnitude among 8 values that is a finite number.
__device__ __forceinline__ float finite_size(u32x4 x, bool bf16) {
  float size = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = fabsf(f16_bits_to_f32(i & 1 ? x[i / 2] >> 16 : x[i / 2] & 0xFFFFu, bf16));
    size = f < __builtin_inff() && f > size ? f : size;
  }
  return size;
}

// A block of positions has one scale for a head: s = max(s of its older positions, max |x| / 448 over its new
// rows), codes the E4M3 values nearest to x / s.  Where s grows, the older codes c become those nearest to
// c (s_old / s).
// A wavefront takes the keys or the values of one block in one head: nobody else touches them, so that the
// codes can be read, scaled and written back without an order among wavefronts.  Its lanes hold the
// new rows' pieces of 8 values (up to 4 each; of larger blocks they are read again for the
// second pass, from the cache).
template <bool RAGGED>
__global__ __launch_bounds__(256) void kv_quantise_kernel(const KvQuantiseArgs A, int bf16) {
  const KvAppendArgs& a = A.a;
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  for (int i = 0; i < kRowLoads; ++i) x[i] = load(min(lane + 64 * i, n - 1));
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int first_slot = begin - in_table * a.page_size;      // of the page
  float* const scale_at = (is_v ? A.v_scale : A.k_scale) + ((int64_t)page * a.Hkv + h) * A.blocks + divided(first_slot, A.by_block);
  const bool older = from > begin;
  const float before = older ? *scale_at : 0.0f;

  float size = 0.0f;
#pragma unroll
  for (int i = 0; i < kRowLoads; ++i) size = fmaxf(size, finite_size(x[i], bf16 != 0));
  for (int i = lane + 64 * kRowLoads; i < n; i += 64) size = fmaxf(size, finite_size(load(i), bf16 != 0));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) size = fmaxf(size, __shfl_xor(size, d));
  const float needed = size / 448.0f;
  const bool grows = older && !(before >= needed);
  const float scale = older && !grows ? before : needed;

  char* const codes = (char*)(is_v ? a.v_cache : a.k_cache) + (int64_t)page * a.page_stride + (int64_t)h * a.head_stride;
  auto code_at = [&](int position, int piece) -> u32x2* {
    return (u32x2*)(codes + (int64_t)(position - in_table * a.page_size) * a.slot_stride + piece * 8);
  };
  if (grows) {
    const float factor = before / scale;
    const int n_old = (from - begin) * pieces;
    for (int i0 = lane; i0 < n_old; i0 += 64 * kOldLoads) {
      u32x2 c[kOldLoads];
#pragma unroll
      for (int j = 0; j < kOldLoads; ++j) {
        const int i = min(i0 + 64 * j, n_old - 1), row = divided(i, a.by_pieces);
        c[j] = *code_at(begin + row, i - row * pieces);
      }
#pragma unroll
      for (int j = 0; j < kOldLoads; ++j) {
        const int i = i0 + 64 * j, row = divided(i, a.by_pieces);
        if (i >= n_old) break;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          typedef __attribute__((ext_vector_type(2))) float f32x2;
          const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j][w], false);
          const f32x2 q = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j][w], true);
          const float f[4] = {p[0] * factor, p[1] * factor, q[0] * factor, q[1] * factor};
          c[j][w] = e4m3x4(f);
        }
        *code_at(begin + row, i - row * pieces) = c[j];
      }
    }
  }
  // (a block of zeros has scale 0, and its codes are zeros)
  const float by = scale > 0.0f ? scale : 1.0f;
#pragma unroll
  for (int i = 0; i < kRowLoads; ++i) {
    const int j = lane + 64 * i, row = divided(j, a.by_pieces);
    if (j < n) *code_at(from + row, j - row * pieces) = e4m3_codes(x[i], by, bf16 != 0);
  }
  for (int j = lane + 64 * kRowLoads; j < n; j += 64) {
    const int row = divided(j, a.by_pieces);
    *code_at(from + row, j - row * pieces) = e4m3_codes(load(j), by, bf16 != 0);
  }
  if (lane == 0 && (grows || !older)) *scale_at = scale;
}

// ---- reading back ----------------------------------------------------------------------------------

// A thread takes the same 8 values of a position's key and value in a head, as the append does.  Bound by the
// rows read and written.
template <bool FP8, bool BF16>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvReadArgs a) {
  const int per_token = a.Hkv * a.pieces;
  const int first = (int)(blockIdx.x * 256 + (threadIdx.x & ~63)), idx = (int)(blockIdx.x * 256 + threadIdx.x);
  if (first >= a.tokens * per_token) return;
  const int t = divided(idx, a.by_token), rest = idx - t * per_token;
  const int h = divided(rest, a.by_pieces), d = (rest - h * a.pieces) * 8;
  const int there = min(t, a.tokens - 1);
  int seq = there;
  bool mine = true;          // the row belongs to a sequence
  if (a.starts != nullptr) {
    const int t0 = divided(first, a.by_token);
    seq = last_not_above(a.B, t0, [&](int i) { return a.starts[i]; });
    while (seq + 1 < a.B && a.starts[seq + 1] <= there) ++seq;
    mine = there >= a.starts[seq] && there < a.starts[seq + 1];
  }
  if (t >= a.tokens) return;
  const int len = a.lens[seq];
  const int pos = a.starts != nullptr ? len - a.starts[seq + 1] + t : len - 1;
  int page = -1, in_table = 0;
  if (mine && pos >= 0 && pos < len) {
    in_table = divided(pos, a.by_page);
    if (in_table < a.table_width) page = a.table[(int64_t)seq * a.table_stride + in_table];
  }
  u32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
  if ((uint32_t)page < (uint32_t)a.num_pages) {
    const int slot = pos - in_table * a.page_size;
    const int64_t from = (int64_t)page * a.page_stride + (int64_t)h * a.head_stride + (int64_t)slot * a.slot_stride + d;
    if constexpr (!FP8) {
      k = *(const u32x4*)((const char*)a.k_cache + from * 2);
      v = *(const u32x4*)((const char*)a.v_cache + from * 2);
    } else {
      const u32x2 kc = *(const u32x2*)((const char*)a.k_cache + from), vc = *(const u32x2*)((const char*)a.v_cache + from);
      const int64_t s = a.blocks == 0 ? h : ((int64_t)page * a.Hkv + h) * a.blocks + divided(slot, a.by_block);
      const float ks = a.k_scale[s], vs = a.v_scale[s];
      typedef __attribute__((ext_vector_type(2))) float f32x2;
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
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x2 k0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)kc[i], false), k1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)kc[i], true);
        const f32x2 v0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vc[i], false), v1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vc[i], true);
        k[2 * i] = pack(k0[0] * ks, k0[1] * ks);
        k[2 * i + 1] = pack(k1[0] * ks, k1[1] * ks);
        v[2 * i] = pack(v0[0] * vs, v0[1] * vs);
        v[2 * i + 1] = pack(v1[0] * vs, v1[1] * vs);
      }
    }
  }
  if (!mine && !a.clear_rest) return;
  *(u32x4*)((char*)a.k + ((int64_t)t * a.k_stride_t + (int64_t)h * a.k_stride_h + d) * 2) = k;
  *(u32x4*)((char*)a.v + ((int64_t)t * a.v_stride_t + (int64_t)h * a.v_stride_h + d) * 2) = v;
}

}  // namespace

void launch_kv_quantise(const KvQuantiseArgs& args, bool bf16, hipStream_t stream) {
  KvQuantiseArgs A = args;
  A.a.pieces = A.a.D / 8;
  A.a.by_page = fast_div(A.a.page_size);
  A.a.by_pieces = fast_div(A.a.pieces);
  A.by_block = fast_div(A.block);
  A.by_heads = fast_div(A.a.Hkv);
  A.slots = (int)kv_quantise_slots(A.a.B, A.a.tokens, A.block, A.a.starts != nullptr);
  const int64_t waves = (int64_t)A.slots * A.a.Hkv * 2;
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
  if (A.a.starts != nullptr)
    hipLaunchKernelGGL((kv_quantise_kernel<true>), grid, block, 0, stream, A, (int)bf16);
  else
    hipLaunchKernelGGL((kv_quantise_kernel<false>), grid, block, 0, stream, A, (int)bf16);
}

void launch_kv_read(const KvReadArgs& args, int kind, hipStream_t stream) {
  KvReadArgs a = args;
  a.pieces = a.D / 8;
  a.by_page = fast_div(a.page_size);
  a.by_pieces = fast_div(a.pieces);
  a.by_token = fast_div(a.Hkv * a.pieces);
  a.by_block = fast_div(a.blocks > 0 ? a.block : 1);
  const int64_t items = (int64_t)a.tokens * a.Hkv * a.pieces;
  const dim3 grid((unsigned)((items + 255) / 256)), block(256);
  const bool fp8 = kind >= 2, b16 = kind % 2 == 0;
  if (!fp8)
    hipLaunchKernelGGL((kv_read_kernel<false, true>), grid, block, 0, stream, a);
  else if (b16)
    hipLaunchKernelGGL((kv_read_kernel<true, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((kv_read_kernel<true, false>), grid, block, 0, stream, a);
}

}  // namespace vk

// kv_blocks.hpp — launchers for 8-bit caches with a scale for each block of positions, and for reading a
// cache back (kv_blocks.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fast_div.hpp"
#include "kv_cache.hpp"

namespace vk {

struct KvQuantiseArgs {
  KvAppendArgs a;           // (its k_scale and v_scale are not used)
  float* k_scale;           // [pages, Hkv, blocks]
  float* v_scale;
  int block, blocks;        // positions of a block, blocks of a page
  // (set by the launcher)
  int slots;
  FastDiv by_block, by_heads;
};
// Places for the blocks of all sequences: those of sequence b begin at starts[b] / block + 2 b.
inline int64_t kv_quantise_slots(int B, int tokens, int block, bool ragged) {
  return ragged ? (int64_t)tokens / block + 2 * (int64_t)B : B;
}
void launch_kv_quantise(const KvQuantiseArgs& a, bool bf16, hipStream_t stream);

struct KvReadArgs {
  const void* k_cache;
  const void* v_cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;    // [B + 1] or null: one row each
  const float* k_scale;     // 8-bit caches: [Hkv] (blocks 0) or [pages, Hkv, blocks]
  const float* v_scale;
  void* k;                  // [tokens, Hkv, D]
  void* v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;   // elements
  int64_t page_stride, head_stride, slot_stride;            // elements
  int table_stride, table_width, num_pages, page_size, block, blocks;
  int B, tokens, Hkv, D;
  bool clear_rest;          // rows that belong to no sequence become zeros
  // (set by the launcher)
  int pieces, chunk;        // 8 values of a row; rows of a workgroup
  FastDiv by_page, by_pieces, by_token, by_block;
};
constexpr int kKvReadChunk = 64;
void launch_kv_read(const KvReadArgs& a, int kind, hipStream_t stream);

}  // namespace vk

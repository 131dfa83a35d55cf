// kv_cache.hpp — launchers of the key-value cache's append and eviction (kv_cache.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "fast_div.hpp"

namespace vk {

struct KvAppendArgs {
  const void* k;            // [tokens, Hkv, D], rows of D values 16-byte aligned
  const void* v;
  void* k_cache;            // [pages, Hkv, page_size, D] by the strides below
  void* v_cache;
  const int32_t* table;     // [B, table_stride]
  const int32_t* lens;      // [B], the new tokens counted
  const int32_t* starts;    // [B + 1] first new token of every sequence, or null: one each
  const float* k_scale;     // [Hkv] (8-bit caches)
  const float* v_scale;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;   // elements
  int64_t page_stride, head_stride, slot_stride;            // elements, of both caches
  int table_stride, table_width, num_pages, page_size;
  int B, tokens, Hkv, D;
  // (set by the launcher)
  int pieces;               // of a row: what a thread takes
  FastDiv by_page, by_pieces, by_token;
};
void launch_kv_append(const KvAppendArgs& a, int kind, hipStream_t stream);

struct KvEvictArgs {
  void* k_cache;            // as above
  void* v_cache;
  const int32_t* table;
  const int32_t* lens;      // [B]
  const float* sums;        // [B, Hkv, sums strides]
  float* sums_out;          // `sums` itself, or another array of its own strides
  int32_t* new_lens;        // [B]
  int32_t* kept;            // [B, Hkv, budget]
  int64_t sums_stride_b, sums_stride_h, out_stride_b, out_stride_h;
  int64_t page_stride, head_stride, slot_stride;            // bytes
  int table_stride, num_pages, page_size, row_bytes;
  int B, Hkv, max_len, budget, keep_first, keep_last;
  uint32_t* order;          // the workspace: for the keys and values of every head a count and a word for
                            // each batch; behind it what the split selection leaves between its launches
  // (set by the launcher)
  uint32_t* split;
  int batches, parts;
  FastDiv by_page, by_pieces;
};
int kv_evict_batches(int budget, int row_bytes);   // of the keys (or values) of a head
constexpr int kKvMoveThreads = 512, kKvMoveFewThreads = 128;   // of a batch's workgroup
size_t kv_evict_workspace_bytes(int rows, int row_bytes, int max_len, int budget);
void launch_kv_evict(const KvEvictArgs& a, hipStream_t stream);

}  // namespace vk

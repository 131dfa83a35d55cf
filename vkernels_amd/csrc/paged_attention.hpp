// paged_attention.hpp — the attention of one new token over a paged key-value cache: the
// kernels' parameters and the sizes that the host and the kernels have to agree on.
// (The kernels are in paged_attention.hip; the entry points in kv_capi.cpp.)
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vk {

// Kinds of cache and query (VK_HIP_KV_* of vkernels_hip.h).
enum KvKind { kKvBf16 = 0, kKvF16 = 1, kKvFp8Bf16 = 2, kKvFp8F16 = 3 };

constexpr int kPaHeads = 16;       // query heads of a work item: the columns of an MFMA tile
constexpr int kPaWaveRows = 32;    // positions a wavefront takes at a time
constexpr int kPaWaves = 4;
constexpr int kPaUnit = kPaWaveRows * kPaWaves;  // positions a workgroup takes at a time

struct PagedAttentionArgs {
  const void* q;            // [B, Hkv * G, D], rows of D values 16-byte aligned
  const void* k_cache;      // [pages, Hkv, page_size, D] by the strides below
  const void* v_cache;
  const int32_t* table;     // [B, table_stride]: the page of every page_size positions
  const int32_t* lens;      // [B]
  const float* sinks;       // [Hkv * G] or null
  const float* k_scale;     // [Hkv] or null; with scale_blocks [pages, Hkv, scale_blocks]
  const float* v_scale;
  void* out;                // [B, Hkv * G, D]
  float* lse;               // [B, Hkv * G] or null
  float* sums;              // [B, Hkv, sums_stride] or null
  void* workspace;
  int64_t q_stride_b, q_stride_h;                       // elements
  int64_t page_stride, head_stride, slot_stride;        // elements, of both caches
  int64_t sums_stride_b, sums_stride_h;                 // elements
  int table_stride, table_width, num_pages, page_size;
  int B, Hkv, G, D, max_len, window;
  int keep_first;           // of a window: positions at the sequence's beginning that stay visible
  int scale_blocks;         // blocks of a page that have a scale of their own (0: one for each head)
  float scale, softcap;
};

// How a call is cut up: the same for the size of the workspace and for the launch.
struct PagedAttentionPlan {
  int head_tiles;           // work items of 16 query heads for each key/value head
  int items;                // B * Hkv * head_tiles
  int workgroups;           // workgroups that share the units evenly; 0: one for each item, whole
  int tile_groups;          // head_tiles, where each tile's items have workgroups of their own; else 1
  int group_workgroups;     // ... so many
  int min_units;            // least share of a workgroup
  int score_pitch;          // positions a row of kept scores is long (0: none are kept)
  size_t ends_at, meta_at, stats_at, ml_at, part_at, scores_at, bytes;  // parts of the workspace
};

PagedAttentionPlan paged_attention_plan(int kind, int B, int Hkv, int G, int D, int max_len, int window, int keep_first,
                                        bool counted);
void launch_paged_attention(const PagedAttentionArgs& a, int kind, hipStream_t stream);

}  // namespace vk

// prompt_attention.hpp — the attention of several new tokens of every sequence over a paged key-value cache: the
// kernels' parameters and how a call is cut up.  (The kernels are in prompt_attention.hip; the entry points
// in kv_capi.cpp.)
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vk {

constexpr int kPromptRows = 128;   // of a workgroup: a row is a query head of a token, the G heads of a key/value
                                   // head and a token one behind the other
constexpr int kPromptFewRows = 32; // ... where sequences have few rows: the wavefronts share the positions instead
constexpr int kPromptFewWidth = 128;   // ... and heads of no more values, or an 8-bit cache
constexpr int kPromptKeys = 64;    // positions a workgroup takes at a time

struct PromptAttentionArgs {
  const void* q;            // [tokens, Hkv * G, D], rows of D values 16-byte aligned
  const void* k_cache;      // [pages, Hkv, page_size, D] by the strides below
  const void* v_cache;
  const int32_t* table;     // [B, table_stride]
  const int32_t* lens;      // [B], the new tokens counted
  const int32_t* starts;    // [B + 1]
  const float* sinks;       // [Hkv * G] or null
  const float* k_scale;     // 8-bit caches: [Hkv], with scale_blocks [pages, Hkv, scale_blocks]
  const float* v_scale;
  void* out;                // [tokens, Hkv * G, D]
  float* lse;               // [tokens, Hkv * G] or null
  void* workspace;
  int64_t q_stride_t, q_stride_h;                       // elements
  int64_t page_stride, head_stride, slot_stride;        // elements, of both caches
  int table_stride, num_pages, page_size, scale_blocks;
  int B, tokens, Hkv, G, D, max_len, window, keep_first;
  float scale, softcap;
  bool clear_rest;          // rows that belong to no sequence become zeros
};

struct PromptAttentionPlan {
  int row_shift;            // a tile has 2^row_shift rows
  int slots;                // places for the tiles of all sequences, and of the rows in front of and behind them
  int splits;               // workgroups that share a tile's positions; more than 1: joined by a second launch
  int share;                // kPromptKeys positions that each of them takes at most
  size_t ml_at, part_at, bytes;   // parts of the workspace
};
int64_t prompt_attention_slots(int B, int tokens, int G, int D, bool fp8);
PromptAttentionPlan prompt_attention_plan(int B, int tokens, int Hkv, int G, int D, int max_len, int window, int keep_first,
                                          bool fp8);
void launch_prompt_attention(const PromptAttentionArgs& a, int kind, hipStream_t stream);

}  // namespace vk

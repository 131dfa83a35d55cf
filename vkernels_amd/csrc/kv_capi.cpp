// kv_capi.cpp — the extern "C" surface of the key-value cache's operators (declared in
// include/vkernels_hip.h): argument checks and error state; the kernels are in
// paged_attention.hip and kv_cache.hip.
#include "vkernels_hip.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "kv_cache.hpp"
#include "paged_attention.hpp"

namespace {

constexpr int64_t kInt32 = 0x7FFFFFFFll;
constexpr int64_t kThreads = 0xFFFFFFFFll;   // of a launch
constexpr int64_t kPositions = kInt32 - (1 << 20);   // positions are ints, a tile or a stretch beyond the last one too

int refuse(int code, const char* who, const char* why) {
  vk_set_last_error(code, (std::string(who) + ": " + why).c_str());
  return code;
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// What every operator asks of the cache: why not, or null.
const char* cache_refusal(const void* k_cache, const void* v_cache, const int32_t* table, const int32_t* lens,
                          int elem, int Hkv, int D, int num_pages, int page_size, int table_width,
                          int table_stride, int64_t page_stride, int64_t head_stride, int64_t slot_stride) {
  if (Hkv <= 0) return "Hkv must be positive";
  if (D <= 0 || D % 16 != 0 || D > 256) return "D must be a multiple of 16 up to 256";
  if (num_pages <= 0 || page_size <= 0) return "num_pages and page_size must be positive";
  if (table_width <= 0 || table_stride < 0) return "block_table must have columns and no negative table_stride";
  if (k_cache == nullptr || v_cache == nullptr || table == nullptr || lens == nullptr)
    return "k_cache/v_cache/block_table/seq_lens must not be null";
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || page_stride * elem % 16 != 0 ||
      head_stride * elem % 16 != 0 || slot_stride * elem % 16 != 0)
    return "rows of the cache must start on 16 bytes";
  if (page_stride < 0 || head_stride < 0 || slot_stride < 0) return "strides must not be negative";
  if (slot_stride > (1ll << 26)) return "slot_stride must be at most 2^26";
  return nullptr;
}

// What is written to holds every element once.
const char* broadcast_refusal(int Hkv, int num_pages, int page_size, int64_t page_stride, int64_t head_stride,
                              int64_t slot_stride) {
  if ((page_stride == 0 && num_pages > 1) || (head_stride == 0 && Hkv > 1) || (slot_stride == 0 && page_size > 1))
    return "a cache that is written to must not be broadcast";
  return nullptr;
}
bool broadcast_sums(int B, int Hkv, int64_t stride_b, int64_t stride_h) {
  return (stride_b == 0 && B > 1) || (stride_h == 0 && Hkv > 1);
}

int launched(const char* who, hipError_t before) {
  const hipError_t err = hipPeekAtLastError();
  if (err == hipSuccess || before != hipSuccess) return VK_OK;
  return refuse(VK_ERROR_INTERNAL, who, hipGetErrorString(err));
}

bool known_kind(int kind) { return kind >= VK_HIP_KV_BF16 && kind <= VK_HIP_KV_FP8_F16; }
int elem_of(int kind) { return kind >= VK_HIP_KV_FP8_BF16 ? 1 : 2; }

}  // namespace

extern "C" {

int vk_hip_kv_cache_append(const void* k, const void* v, void* k_cache, void* v_cache,
                           const int32_t* block_table, const int32_t* seq_lens,
                           const int32_t* query_start, const float* k_scale, const float* v_scale,
                           int kind, int B, int tokens, int Hkv, int D, int num_pages, int page_size,
                           int table_width, int table_stride, int64_t k_stride_t, int64_t k_stride_h,
                           int64_t v_stride_t, int64_t v_stride_h, int64_t page_stride,
                           int64_t head_stride, int64_t slot_stride, void* stream) {
  const char* const who = "vk_hip_kv_cache_append";
  if (!known_kind(kind)) return refuse(VK_ERROR_UNSUPPORTED, who, "kind must be one of VK_HIP_KV_*");
  if (B < 0 || tokens < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "B and tokens must not be negative");
  if (query_start == nullptr && tokens != B)
    return refuse(VK_ERROR_INVALID_ARGUMENT, who, "without query_start there is one token for each sequence");
  if (tokens == 0 || B == 0) return VK_OK;
  const char* why = cache_refusal(k_cache, v_cache, block_table, seq_lens, elem_of(kind), Hkv, D, num_pages, page_size,
                                  table_width, table_stride, page_stride, head_stride, slot_stride);
  if (why == nullptr) why = broadcast_refusal(Hkv, num_pages, page_size, page_stride, head_stride, slot_stride);
  if (why == nullptr && (k == nullptr || v == nullptr)) why = "k/v must not be null";
  if (why == nullptr && (!aligned(k, 16) || !aligned(v, 16) || k_stride_t % 8 != 0 || k_stride_h % 8 != 0 ||
                         v_stride_t % 8 != 0 || v_stride_h % 8 != 0))
    why = "rows of k and v must start on 16 bytes";
  if (why == nullptr && elem_of(kind) == 1 && (k_scale == nullptr || v_scale == nullptr))
    why = "an 8-bit cache needs k_scale and v_scale";
  if (why == nullptr && elem_of(kind) == 2 && (k_scale != nullptr || v_scale != nullptr))
    why = "k_scale and v_scale are for 8-bit caches";
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  if ((int64_t)tokens * Hkv > kInt32 / D) return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many values for one call");
  vk::KvAppendArgs a{};
  a.k = k; a.v = v; a.k_cache = k_cache; a.v_cache = v_cache; a.table = block_table; a.lens = seq_lens;
  a.starts = query_start; a.k_scale = k_scale; a.v_scale = v_scale;
  a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h; a.v_stride_t = v_stride_t; a.v_stride_h = v_stride_h;
  a.page_stride = page_stride; a.head_stride = head_stride; a.slot_stride = slot_stride;
  a.table_stride = table_stride; a.table_width = table_width; a.num_pages = num_pages; a.page_size = page_size;
  a.B = B; a.tokens = tokens; a.Hkv = Hkv; a.D = D;
  const hipError_t before = hipPeekAtLastError();
  vk::launch_kv_append(a, kind, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

size_t vk_hip_paged_attention_workspace_bytes(int kind, int B, int Hkv, int G, int D, int max_len, int window,
                                              int counted) {
  if (!known_kind(kind) || B <= 0 || Hkv <= 0 || G <= 0 || D <= 0 || max_len < 0) return 0;
  return vk::paged_attention_plan(kind, B, Hkv, G, D, max_len, window, counted != 0).bytes;
}

int vk_hip_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                           const int32_t* block_table, const int32_t* seq_lens, const float* sinks,
                           const float* k_scale, const float* v_scale, void* out, float* lse,
                           float* weight_sums, int kind, int B, int Hkv, int G, int D, int num_pages,
                           int page_size, int table_width, int table_stride, int max_len, int window,
                           float scale, float softcap, int64_t q_stride_b, int64_t q_stride_h,
                           int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                           int64_t sums_stride_b, int64_t sums_stride_h, void* workspace,
                           size_t workspace_bytes, void* stream) {
  const char* const who = "vk_hip_paged_attention";
  if (!known_kind(kind)) return refuse(VK_ERROR_UNSUPPORTED, who, "kind must be one of VK_HIP_KV_*");
  if (B < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "B must not be negative");
  if (B == 0) return VK_OK;
  const char* why = cache_refusal(k_cache, v_cache, block_table, seq_lens, elem_of(kind), Hkv, D, num_pages, page_size,
                                  table_width, table_stride, page_stride, head_stride, slot_stride);
  if (why == nullptr && G <= 0) why = "G must be positive";
  if (why == nullptr && (q == nullptr || out == nullptr)) why = "q/out must not be null";
  if (why == nullptr && (!aligned(q, 16) || !aligned(out, 16) || q_stride_b % 8 != 0 || q_stride_h % 8 != 0))
    why = "rows of q and out must start on 16 bytes";
  if (why == nullptr && (max_len < 0 || max_len > (int64_t)table_width * page_size))
    why = "max_len must be within the table's positions";
  if (why == nullptr && weight_sums != nullptr && broadcast_sums(B, Hkv, sums_stride_b, sums_stride_h))
    why = "weight_sums must not be broadcast";
  if (why == nullptr && !(softcap >= 0.0f)) why = "softcap must not be negative";
  if (why == nullptr && elem_of(kind) == 2 && (k_scale != nullptr || v_scale != nullptr))
    why = "k_scale and v_scale are for 8-bit caches";
  if (why == nullptr && elem_of(kind) == 1 && (k_scale == nullptr || v_scale == nullptr))
    why = "an 8-bit cache needs k_scale and v_scale";
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  // (units of work are counted in 32 bits, and so are a launch's threads, 256 for each item or chunk)
  const int64_t rows = (int64_t)B * Hkv, items = rows * ((G + vk::kPaHeads - 1) / vk::kPaHeads);
  if (max_len > kPositions || rows > kInt32 / G || items > kThreads / 512 || items > kInt32 / (max_len / vk::kPaUnit + 3) / 2 ||
      rows > kThreads / 512 / (max_len / 4096 + 2))
    return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many sequences, heads and positions for one call");
  const vk::PagedAttentionPlan plan = vk::paged_attention_plan(kind, B, Hkv, G, D, max_len, window, weight_sums != nullptr);
  if (plan.bytes > 0 && (workspace == nullptr || workspace_bytes < plan.bytes || !aligned(workspace, 16)))
    return refuse(VK_ERROR_INVALID_ARGUMENT, who,
                  "a workspace of vk_hip_paged_attention_workspace_bytes (16-byte aligned) is needed");
  vk::PagedAttentionArgs a{};
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.table = block_table; a.lens = seq_lens;
  a.sinks = sinks; a.k_scale = k_scale; a.v_scale = v_scale; a.out = out; a.lse = lse; a.sums = weight_sums;
  a.workspace = workspace;
  a.q_stride_b = q_stride_b; a.q_stride_h = q_stride_h;
  a.page_stride = page_stride; a.head_stride = head_stride; a.slot_stride = slot_stride;
  a.sums_stride_b = sums_stride_b; a.sums_stride_h = sums_stride_h;
  a.table_stride = table_stride; a.table_width = table_width; a.num_pages = num_pages; a.page_size = page_size;
  a.B = B; a.Hkv = Hkv; a.G = G; a.D = D; a.max_len = max_len; a.window = window;
  // (Caps that no score comes near, infinity among them, are none, and below the other bound all scores are alike:
  // the kernel's factors 1 / cap and cap then stay within 32-bit floats.)
  a.scale = scale; a.softcap = softcap >= 0x1p100f ? 0.0f : softcap > 0.0f ? std::fmax(softcap, 0x1p-100f) : 0.0f;
  const hipError_t before = hipPeekAtLastError();
  vk::launch_paged_attention(a, kind, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

size_t vk_hip_kv_cache_evict_workspace_bytes(int elem_bytes, int B, int Hkv, int D, int max_len, int budget) {
  if (elem_bytes <= 0 || B <= 0 || Hkv <= 0 || D < 16 || budget <= 0 || D * (int64_t)elem_bytes > 512) return 0;
  if (static_cast<int64_t>(B) * Hkv > kInt32) return 0;
  return vk::kv_evict_workspace_bytes(B * Hkv, D * elem_bytes, max_len, budget);
}

int vk_hip_kv_cache_evict(void* k_cache, void* v_cache, const int32_t* block_table,
                          const int32_t* seq_lens, const float* weight_sums, float* sums_out,
                          int32_t* new_lens, int32_t* kept, int elem_bytes, int B, int Hkv, int D,
                          int num_pages, int page_size, int table_width, int table_stride, int max_len,
                          int budget, int keep_first, int keep_last, int64_t page_stride,
                          int64_t head_stride, int64_t slot_stride, int64_t sums_stride_b,
                          int64_t sums_stride_h, int64_t out_stride_b, int64_t out_stride_h, void* workspace,
                          size_t workspace_bytes, void* stream) {
  const char* const who = "vk_hip_kv_cache_evict";
  if (elem_bytes != 1 && elem_bytes != 2) return refuse(VK_ERROR_UNSUPPORTED, who, "elem_bytes must be 1 or 2");
  if (B < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "B must not be negative");
  if (B == 0) return VK_OK;
  const char* why = cache_refusal(k_cache, v_cache, block_table, seq_lens, elem_bytes, Hkv, D, num_pages, page_size,
                                  table_width, table_stride, page_stride, head_stride, slot_stride);
  if (why == nullptr) why = broadcast_refusal(Hkv, num_pages, page_size, page_stride, head_stride, slot_stride);
  if (why == nullptr && (weight_sums == nullptr || sums_out == nullptr || new_lens == nullptr || kept == nullptr))
    why = "weight_sums/sums_out/new_lens/kept must not be null";
  if (why == nullptr && (max_len < 0 || max_len > (int64_t)table_width * page_size))
    why = "max_len must be within the table's positions";
  if (why == nullptr && (budget <= 0 || keep_first < 0 || keep_last < 0 || (int64_t)keep_first + keep_last > budget))
    why = "budget must be positive, keep_first and keep_last not negative and their sum within budget";
  if (why == nullptr && sums_out == weight_sums && (out_stride_b != sums_stride_b || out_stride_h != sums_stride_h))
    why = "sums_out in place has weight_sums' strides";
  if (why == nullptr && broadcast_sums(B, Hkv, out_stride_b, out_stride_h)) why = "sums_out must not be broadcast";
  if (why == nullptr && new_lens == seq_lens) why = "new_lens must not be seq_lens";
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  if (max_len > kPositions || (int64_t)B * Hkv > kInt32 / 2 || (int64_t)budget * D * elem_bytes / 16 > kInt32 / 2 ||
      (int64_t)B * Hkv * vk::kv_evict_batches(budget, D * elem_bytes) > kThreads / 2 / vk::kKvMoveThreads)
    return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many rows for one call");
  if (workspace == nullptr || !aligned(workspace, 16) ||
      workspace_bytes < vk_hip_kv_cache_evict_workspace_bytes(elem_bytes, B, Hkv, D, max_len, budget))
    return refuse(VK_ERROR_INVALID_ARGUMENT, who, "a workspace of vk_hip_kv_cache_evict_workspace_bytes is needed");
  vk::KvEvictArgs a{};
  a.k_cache = k_cache; a.v_cache = v_cache; a.table = block_table; a.lens = seq_lens;
  a.sums = weight_sums; a.sums_out = sums_out; a.new_lens = new_lens; a.kept = kept;
  a.sums_stride_b = sums_stride_b; a.sums_stride_h = sums_stride_h;
  a.out_stride_b = out_stride_b; a.out_stride_h = out_stride_h;
  a.page_stride = page_stride * elem_bytes; a.head_stride = head_stride * elem_bytes;
  a.slot_stride = slot_stride * elem_bytes;
  a.table_stride = table_stride; a.num_pages = num_pages; a.page_size = page_size; a.row_bytes = D * elem_bytes;
  a.B = B; a.Hkv = Hkv; a.max_len = max_len; a.budget = budget; a.keep_first = keep_first; a.keep_last = keep_last;
  a.order = static_cast<uint32_t*>(workspace);
  const hipError_t before = hipPeekAtLastError();
  vk::launch_kv_evict(a, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

}  // extern "C"

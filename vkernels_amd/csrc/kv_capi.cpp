// kv_capi.cpp — the extern "C" surface of the key-value cache's operators (declared in
// include/vkernels_hip.h): argument checks and error state; the kernels are in
// kv_cache.hip, kv_blocks.hip, paged_attention.hip, prompt_attention.hip and qk_norm_rope.hip.
#include "vkernels_hip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "kv_blocks.hpp"
#include "kv_cache.hpp"
#include "paged_attention.hpp"
#include "prompt_attention.hpp"
#include "qk_norm_rope.hpp"

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

const char* rows_refusal(const void* k, const void* v, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                         int64_t v_stride_h) {
  if (!aligned(k, 16) || !aligned(v, 16) || k_stride_t % 8 != 0 || k_stride_h % 8 != 0 || v_stride_t % 8 != 0 ||
      v_stride_h % 8 != 0)
    return "rows of k and v must start on 16 bytes";
  return nullptr;
}

// Rows of D values that are written to: heads one behind the other within tokens, or tokens within heads.
bool rows_overlap(int tokens, int heads, int D, int64_t by_t, int64_t by_h) {
  if (by_t < 0 || by_h < 0) return true;
  if (tokens <= 1 || heads <= 1) return (tokens > 1 && by_t < D) || (heads > 1 && by_h < D);
  const bool heads_inside = by_h <= by_t;
  const int64_t inner = heads_inside ? by_h : by_t, outer = heads_inside ? by_t : by_h, n = heads_inside ? heads : tokens;
  return inner < D || outer / inner < n - 1 || outer - inner * (n - 1) < D;
}

const char* scales_refusal(int kind, const float* k_scale, const float* v_scale, int scale_blocks, int page_size) {
  if (elem_of(kind) == 1 && (k_scale == nullptr || v_scale == nullptr)) return "an 8-bit cache needs k_scale and v_scale";
  if (elem_of(kind) == 2 && (k_scale != nullptr || v_scale != nullptr)) return "k_scale and v_scale are for 8-bit caches";
  if (scale_blocks < 0 || (scale_blocks > 0 && (elem_of(kind) == 2 || page_size % scale_blocks != 0)))
    return "blocks with a scale of their own are equal parts of an 8-bit cache's pages";
  return nullptr;
}

// New rows into the cache: with scale_blocks > 0 their scales are the call's own.
int append(const char* who, const void* k, const void* v, void* k_cache, void* v_cache, const int32_t* block_table,
           const int32_t* seq_lens, const int32_t* query_start, float* k_scale, float* v_scale, int scale_blocks, int kind,
           int B, int tokens, int Hkv, int D, int num_pages, int page_size, int table_width, int table_stride,
           int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, int64_t page_stride,
           int64_t head_stride, int64_t slot_stride, void* stream) {
  if (!known_kind(kind)) return refuse(VK_ERROR_UNSUPPORTED, who, "kind must be one of VK_HIP_KV_*");
  if (B < 0 || tokens < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "B and tokens must not be negative");
  if (query_start == nullptr && tokens != B)
    return refuse(VK_ERROR_INVALID_ARGUMENT, who, "without query_start there is one token for each sequence");
  if (tokens == 0 || B == 0) return VK_OK;
  const char* why = cache_refusal(k_cache, v_cache, block_table, seq_lens, elem_of(kind), Hkv, D, num_pages, page_size,
                                  table_width, table_stride, page_stride, head_stride, slot_stride);
  if (why == nullptr) why = broadcast_refusal(Hkv, num_pages, page_size, page_stride, head_stride, slot_stride);
  if (why == nullptr && (k == nullptr || v == nullptr)) why = "k/v must not be null";
  if (why == nullptr) why = rows_refusal(k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h);
  if (why == nullptr) why = scales_refusal(kind, k_scale, v_scale, scale_blocks, page_size);
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  if ((int64_t)tokens * Hkv > kInt32 / D) return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many values for one call");
  vk::KvAppendArgs a{};
  a.k = k; a.v = v; a.k_cache = k_cache; a.v_cache = v_cache; a.table = block_table; a.lens = seq_lens;
  a.starts = query_start; a.k_scale = k_scale; a.v_scale = v_scale;
  a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h; a.v_stride_t = v_stride_t; a.v_stride_h = v_stride_h;
  a.page_stride = page_stride; a.head_stride = head_stride; a.slot_stride = slot_stride;
  a.table_stride = table_stride; a.table_width = table_width; a.num_pages = num_pages; a.page_size = page_size;
  a.B = B; a.tokens = tokens; a.Hkv = Hkv; a.D = D;
  if (scale_blocks > 0) {
    vk::KvQuantiseArgs A{};
    A.a = a;
    A.k_scale = k_scale; A.v_scale = v_scale; A.blocks = scale_blocks; A.block = page_size / scale_blocks;
    if (vk::kv_quantise_slots(B, tokens, A.block, query_start != nullptr) > kThreads / 512 / 2 / Hkv)
      return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many values for one call");
    const hipError_t before = hipPeekAtLastError();
    vk::launch_kv_quantise(A, kind == VK_HIP_KV_FP8_BF16, static_cast<hipStream_t>(stream));
    return launched(who, before);
  }
  const hipError_t before = hipPeekAtLastError();
  vk::launch_kv_append(a, kind, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

// Caps that no score comes near, infinity among them, are none, and below the other bound all scores are alike:
// the kernels' factors 1 / cap and cap then stay within 32-bit floats.
float cap_of(float softcap) { return softcap >= 0x1p100f ? 0.0f : softcap > 0.0f ? std::fmax(softcap, 0x1p-100f) : 0.0f; }

// Rows and slots are counted in 32 bits, and so are a launch's threads.  (Where tiles are shared there are few: at most
// 4096 workgroups and one for every head more.)
bool prompt_fits(int B, int tokens, int Hkv, int G, int D) {
  if (tokens > kInt32 / 4 / G || B > kInt32 / 4) return false;
  return vk::prompt_attention_slots(B, tokens, G, D, true) <= kThreads / 512 / Hkv;      // (in smaller tiles, if the cache's type says so)
}

// Attention of one new token of every sequence.
int attend(const char* who, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
           const int32_t* seq_lens, const float* sinks, const float* k_scale, const float* v_scale, int scale_blocks,
           void* out, float* lse, float* weight_sums, int kind, int B, int Hkv, int G, int D, int num_pages, int page_size,
           int table_width, int table_stride, int max_len, int window, int keep_first, float scale, float softcap,
           int64_t q_stride_b, int64_t q_stride_h, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
           int64_t sums_stride_b, int64_t sums_stride_h, void* workspace, size_t workspace_bytes, void* stream) {
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
  if (why == nullptr && keep_first < 0) why = "keep_first must not be negative";
  if (why == nullptr) why = scales_refusal(kind, k_scale, v_scale, scale_blocks, page_size);
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  // (units of work are counted in 32 bits, and so are a launch's threads, 256 for each item or chunk)
  const int64_t rows = (int64_t)B * Hkv, items = rows * ((G + vk::kPaHeads - 1) / vk::kPaHeads);
  if (max_len > kPositions || rows > kInt32 / G || items > kThreads / 512 || items > kInt32 / (max_len / vk::kPaUnit + 3) / 2 ||
      rows > kThreads / 512 / (max_len / 4096 + 2))
    return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many sequences, heads and positions for one call");
  const vk::PagedAttentionPlan plan = vk::paged_attention_plan(kind, B, Hkv, G, D, max_len, window, keep_first, weight_sums != nullptr);
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
  a.keep_first = window > 0 ? keep_first : 0; a.scale_blocks = scale_blocks;
  a.scale = scale; a.softcap = cap_of(softcap);
  const hipError_t before = hipPeekAtLastError();
  vk::launch_paged_attention(a, kind, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

}  // namespace

extern "C" {

int vk_hip_kv_cache_append(const void* k, const void* v, void* k_cache, void* v_cache,
                           const int32_t* block_table, const int32_t* seq_lens,
                           const int32_t* query_start, const float* k_scale, const float* v_scale,
                           int kind, int B, int tokens, int Hkv, int D, int num_pages, int page_size,
                           int table_width, int table_stride, int64_t k_stride_t, int64_t k_stride_h,
                           int64_t v_stride_t, int64_t v_stride_h, int64_t page_stride,
                           int64_t head_stride, int64_t slot_stride, void* stream) {
  return append("vk_hip_kv_cache_append", k, v, k_cache, v_cache, block_table, seq_lens, query_start, const_cast<float*>(k_scale),
                const_cast<float*>(v_scale), 0, kind, B, tokens, Hkv, D, num_pages, page_size, table_width, table_stride,
                k_stride_t, k_stride_h, v_stride_t, v_stride_h, page_stride, head_stride, slot_stride, stream);
}

int vk_hip_kv_cache_append_ex(const void* k, const void* v, void* k_cache, void* v_cache,
                              const int32_t* block_table, const int32_t* seq_lens,
                              const int32_t* query_start, float* k_scale, float* v_scale, int scale_blocks,
                              int kind, int B, int tokens, int Hkv, int D, int num_pages, int page_size,
                              int table_width, int table_stride, int64_t k_stride_t, int64_t k_stride_h,
                              int64_t v_stride_t, int64_t v_stride_h, int64_t page_stride,
                              int64_t head_stride, int64_t slot_stride, void* stream) {
  return append("vk_hip_kv_cache_append_ex", k, v, k_cache, v_cache, block_table, seq_lens, query_start, k_scale, v_scale,
                scale_blocks, kind, B, tokens, Hkv, D, num_pages, page_size, table_width, table_stride, k_stride_t, k_stride_h,
                v_stride_t, v_stride_h, page_stride, head_stride, slot_stride, stream);
}

int vk_hip_kv_cache_read(const void* k_cache, const void* v_cache, const int32_t* block_table,
                         const int32_t* seq_lens, const int32_t* query_start, const float* k_scale,
                         const float* v_scale, int scale_blocks, void* k, void* v, int kind, int B, int tokens,
                         int Hkv, int D, int num_pages, int page_size, int table_width, int table_stride,
                         int clear_rest, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                         int64_t v_stride_h, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                         void* stream) {
  const char* const who = "vk_hip_kv_cache_read";
  if (!known_kind(kind)) return refuse(VK_ERROR_UNSUPPORTED, who, "kind must be one of VK_HIP_KV_*");
  if (B < 0 || tokens < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "B and tokens must not be negative");
  if (query_start == nullptr && tokens != B)
    return refuse(VK_ERROR_INVALID_ARGUMENT, who, "without query_start there is one token for each sequence");
  if (tokens == 0) return VK_OK;
  if (B == 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "rows need a sequence to be read from");
  const char* why = cache_refusal(k_cache, v_cache, block_table, seq_lens, elem_of(kind), Hkv, D, num_pages, page_size,
                                  table_width, table_stride, page_stride, head_stride, slot_stride);
  if (why == nullptr && (k == nullptr || v == nullptr)) why = "k/v must not be null";
  if (why == nullptr) why = rows_refusal(k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h);
  if (why == nullptr && (rows_overlap(tokens, Hkv, D, k_stride_t, k_stride_h) || rows_overlap(tokens, Hkv, D, v_stride_t, v_stride_h)))
    why = "rows of k and v must not overlap";
  if (why == nullptr) why = scales_refusal(kind, k_scale, v_scale, scale_blocks, page_size);
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  if ((int64_t)tokens * Hkv > kInt32 / D || tokens > kThreads / 512)
    return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many values for one call");
  vk::KvReadArgs a{};
  a.k_cache = k_cache; a.v_cache = v_cache; a.table = block_table; a.lens = seq_lens; a.starts = query_start;
  a.k_scale = k_scale; a.v_scale = v_scale; a.k = k; a.v = v;
  a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h; a.v_stride_t = v_stride_t; a.v_stride_h = v_stride_h;
  a.page_stride = page_stride; a.head_stride = head_stride; a.slot_stride = slot_stride;
  a.table_stride = table_stride; a.table_width = table_width; a.num_pages = num_pages; a.page_size = page_size;
  a.blocks = scale_blocks; a.block = scale_blocks > 0 ? page_size / scale_blocks : 0;
  a.B = B; a.tokens = tokens; a.Hkv = Hkv; a.D = D; a.clear_rest = clear_rest != 0;
  const hipError_t before = hipPeekAtLastError();
  vk::launch_kv_read(a, kind, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

size_t vk_hip_paged_attention_workspace_bytes(int kind, int B, int Hkv, int G, int D, int max_len, int window,
                                              int counted) {
  return vk_hip_paged_attention_workspace_bytes_ex(kind, B, Hkv, G, D, max_len, window, 0, counted);
}

size_t vk_hip_paged_attention_workspace_bytes_ex(int kind, int B, int Hkv, int G, int D, int max_len, int window,
                                                 int keep_first, int counted) {
  if (!known_kind(kind) || B <= 0 || Hkv <= 0 || G <= 0 || D <= 0 || max_len < 0 || keep_first < 0) return 0;
  return vk::paged_attention_plan(kind, B, Hkv, G, D, max_len, window, keep_first, counted != 0).bytes;
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
  return attend("vk_hip_paged_attention", q, k_cache, v_cache, block_table, seq_lens, sinks, k_scale, v_scale, 0, out, lse,
                weight_sums, kind, B, Hkv, G, D, num_pages, page_size, table_width, table_stride, max_len, window, 0, scale,
                softcap, q_stride_b, q_stride_h, page_stride, head_stride, slot_stride, sums_stride_b, sums_stride_h,
                workspace, workspace_bytes, stream);
}

int vk_hip_paged_attention_ex(const void* q, const void* k_cache, const void* v_cache,
                              const int32_t* block_table, const int32_t* seq_lens, const float* sinks,
                              const float* k_scale, const float* v_scale, int scale_blocks, void* out, float* lse,
                              float* weight_sums, int kind, int B, int Hkv, int G, int D, int num_pages,
                              int page_size, int table_width, int table_stride, int max_len, int window,
                              int keep_first, float scale, float softcap, int64_t q_stride_b, int64_t q_stride_h,
                              int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                              int64_t sums_stride_b, int64_t sums_stride_h, void* workspace,
                              size_t workspace_bytes, void* stream) {
  return attend("vk_hip_paged_attention_ex", q, k_cache, v_cache, block_table, seq_lens, sinks, k_scale, v_scale, scale_blocks,
                out, lse, weight_sums, kind, B, Hkv, G, D, num_pages, page_size, table_width, table_stride, max_len, window,
                keep_first, scale, softcap, q_stride_b, q_stride_h, page_stride, head_stride, slot_stride, sums_stride_b,
                sums_stride_h, workspace, workspace_bytes, stream);
}

size_t vk_hip_paged_attention_prompt_workspace_bytes(int B, int tokens, int Hkv, int G, int D, int max_len, int window,
                                                     int keep_first) {
  if (B <= 0 || tokens <= 0 || Hkv <= 0 || G <= 0 || D <= 0 || max_len < 0 || keep_first < 0) return 0;
  if (!prompt_fits(B, tokens, Hkv, G, D)) return 0;
  auto bytes = [&](bool fp8) {
    return vk::prompt_attention_plan(B, tokens, Hkv, G, D, max_len, window, window > 0 ? keep_first : 0, fp8).bytes;
  };
  return std::max(bytes(false), bytes(true));      // (a cache of either type)
}

int vk_hip_paged_attention_prompt(const void* q, const void* k_cache, const void* v_cache,
                                  const int32_t* block_table, const int32_t* seq_lens, const int32_t* query_start,
                                  const float* sinks, const float* k_scale, const float* v_scale, int scale_blocks,
                                  void* out, float* lse, int kind, int B, int tokens, int Hkv, int G, int D,
                                  int num_pages, int page_size, int table_width, int table_stride, int max_len,
                                  int window, int keep_first, int clear_rest, float scale, float softcap,
                                  int64_t q_stride_t, int64_t q_stride_h, int64_t page_stride, int64_t head_stride,
                                  int64_t slot_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* const who = "vk_hip_paged_attention_prompt";
  if (!known_kind(kind)) return refuse(VK_ERROR_UNSUPPORTED, who, "kind must be one of VK_HIP_KV_*");
  if (B < 0 || tokens < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "B and tokens must not be negative");
  if (tokens == 0) return VK_OK;
  if (B == 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "tokens need a sequence");
  const char* why = cache_refusal(k_cache, v_cache, block_table, seq_lens, elem_of(kind), Hkv, D, num_pages, page_size,
                                  table_width, table_stride, page_stride, head_stride, slot_stride);
  if (why == nullptr && G <= 0) why = "G must be positive";
  if (why == nullptr && (q == nullptr || out == nullptr || query_start == nullptr)) why = "q/out/query_start must not be null";
  if (why == nullptr && (!aligned(q, 16) || !aligned(out, 16) || q_stride_t % 8 != 0 || q_stride_h % 8 != 0))
    why = "rows of q and out must start on 16 bytes";
  if (why == nullptr && (max_len < 0 || max_len > (int64_t)table_width * page_size))
    why = "max_len must be within the table's positions";
  if (why == nullptr && keep_first < 0) why = "keep_first must not be negative";
  if (why == nullptr && !(softcap >= 0.0f)) why = "softcap must not be negative";
  if (why == nullptr) why = scales_refusal(kind, k_scale, v_scale, scale_blocks, page_size);
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  if (max_len > kPositions || !prompt_fits(B, tokens, Hkv, G, D))
    return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many sequences, tokens, heads and positions for one call");
  keep_first = window > 0 ? keep_first : 0;
  const vk::PromptAttentionPlan plan = vk::prompt_attention_plan(B, tokens, Hkv, G, D, max_len, window, keep_first, elem_of(kind) == 1);
  if (plan.bytes > 0 && (workspace == nullptr || workspace_bytes < plan.bytes || !aligned(workspace, 16)))
    return refuse(VK_ERROR_INVALID_ARGUMENT, who,
                  "a workspace of vk_hip_paged_attention_prompt_workspace_bytes (16-byte aligned) is needed");
  vk::PromptAttentionArgs a{};
  a.q = q; a.k_cache = k_cache; a.v_cache = v_cache; a.table = block_table; a.lens = seq_lens; a.starts = query_start;
  a.sinks = sinks; a.k_scale = k_scale; a.v_scale = v_scale; a.out = out; a.lse = lse; a.workspace = workspace;
  a.q_stride_t = q_stride_t; a.q_stride_h = q_stride_h;
  a.page_stride = page_stride; a.head_stride = head_stride; a.slot_stride = slot_stride;
  a.table_stride = table_stride; a.num_pages = num_pages; a.page_size = page_size; a.scale_blocks = scale_blocks;
  a.B = B; a.tokens = tokens; a.Hkv = Hkv; a.G = G; a.D = D; a.max_len = max_len; a.window = window; a.keep_first = keep_first;
  a.scale = scale; a.softcap = cap_of(softcap); a.clear_rest = clear_rest != 0;
  const hipError_t before = hipPeekAtLastError();
  vk::launch_prompt_attention(a, kind, static_cast<hipStream_t>(stream));
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

int vk_hip_qk_norm_rope(const void* q, const void* k, const int32_t* positions, const float* inv_freq,
                        const void* q_weight, const void* k_weight, void* q_out, void* k_out, int kind,
                        int weights_f32, int T, int Hq, int Hkv, int D, int turned, int pairs, int axes,
                        const int32_t* sections, int norm, float eps, float factor, int64_t q_stride_t,
                        int64_t q_stride_h, int64_t k_stride_t, int64_t k_stride_h, int64_t q_out_stride_t,
                        int64_t q_out_stride_h, int64_t k_out_stride_t, int64_t k_out_stride_h,
                        int64_t axis_stride, void* stream) {
  const char* const who = "vk_hip_qk_norm_rope";
  if (kind != VK_HIP_KV_BF16 && kind != VK_HIP_KV_F16)
    return refuse(VK_ERROR_UNSUPPORTED, who, "kind must be VK_HIP_KV_BF16 or VK_HIP_KV_F16");
  if (T < 0) return refuse(VK_ERROR_INVALID_ARGUMENT, who, "T must not be negative");
  if (T == 0) return VK_OK;
  const char* why = nullptr;
  if (Hq <= 0 || Hkv <= 0) why = "Hq and Hkv must be positive";
  if (why == nullptr && (D <= 0 || D % 16 != 0 || D > 256)) why = "D must be a multiple of 16 up to 256";
  if (why == nullptr && (turned <= 0 || turned % 8 != 0 || turned > D))
    why = "the values that are rotated must be a multiple of 8 up to D";
  if (why == nullptr && (axes <= 0 || axes > vk::kRopeAxes)) why = "there are 1 to 4 axes";
  if (why == nullptr && axes > 1 && sections == nullptr) why = "several axes need sections";
  if (why == nullptr && (q == nullptr || k == nullptr || q_out == nullptr || k_out == nullptr || positions == nullptr ||
                         inv_freq == nullptr))
    why = "q/k/q_out/k_out/positions/inv_freq must not be null";
  if (why == nullptr && !norm && (q_weight != nullptr || k_weight != nullptr)) why = "weights belong to the norm";
  if (why == nullptr && norm && !(eps >= 0.0f)) why = "eps must not be negative";
  if (why == nullptr && (!aligned(q_weight, 16) || !aligned(k_weight, 16))) why = "weights must start on 16 bytes";
  if (why == nullptr && (!aligned(q, 16) || !aligned(k, 16) || !aligned(q_out, 16) || !aligned(k_out, 16) ||
                         (q_stride_t | q_stride_h | k_stride_t | k_stride_h | q_out_stride_t | q_out_stride_h |
                          k_out_stride_t | k_out_stride_h) % 8 != 0))
    why = "rows of q, k and the results must start on 16 bytes";
  if (why == nullptr && (q_stride_t < 0 || q_stride_h < 0 || k_stride_t < 0 || k_stride_h < 0 || axis_stride < 0))
    why = "strides must not be negative";
  if (why == nullptr && (rows_overlap(T, Hq, D, q_out_stride_t, q_out_stride_h) ||
                         rows_overlap(T, Hkv, D, k_out_stride_t, k_out_stride_h)))
    why = "rows of the results must not overlap";
  vk::QkNormRopeArgs a{};
  a.section_end[0] = turned / 2;
  int64_t all = 0;
  for (int i = 0; why == nullptr && axes > 1 && i < axes; ++i) {
    if (sections[i] < 0) why = "sections must not be negative";
    all += sections[i];
    a.section_end[i] = (int)(all < turned ? all : turned);
  }
  if (why == nullptr && axes > 1 && all != turned / 2) why = "sections must add up to half the values that are rotated";
  if (why != nullptr) return refuse(VK_ERROR_INVALID_ARGUMENT, who, why);
  if (T > kThreads / 256 || Hq > kInt32 / 2 || Hkv > kInt32 / 2 - 4096)
    return refuse(VK_ERROR_OUT_OF_RANGE, who, "too many tokens or heads for one call");
  a.q = q; a.k = k; a.q_out = q_out; a.k_out = k_out; a.q_weight = q_weight; a.k_weight = k_weight;
  a.positions = positions; a.inv_freq = inv_freq;
  a.q_stride_t = q_stride_t; a.q_stride_h = q_stride_h; a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h;
  a.qo_stride_t = q_out_stride_t; a.qo_stride_h = q_out_stride_h;
  a.ko_stride_t = k_out_stride_t; a.ko_stride_h = k_out_stride_h;
  a.axis_stride = axis_stride;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.turned = turned; a.axes = axes;
  a.eps = eps; a.factor = factor; a.norm = norm != 0; a.weights_f32 = weights_f32 != 0;
  const hipError_t before = hipPeekAtLastError();
  vk::launch_qk_norm_rope(a, kind == VK_HIP_KV_BF16, pairs != 0, static_cast<hipStream_t>(stream));
  return launched(who, before);
}

}  // extern "C"

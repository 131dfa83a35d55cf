// kv_cache.hip — new rows into a paged key-value cache, and its eviction by accumulated
// attention weight: the positions of most weight are selected and the cache is compacted
// to them, in place.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_cache.hpp"
#include "paged_attention.hpp"

namespace vk {
namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// ---- append --------------------------------------------------------------------------------

// The largest of 64-bit-scaled E4M3: what does not fit is stored as the largest finite code.
__device__ __forceinline__ float e4m3_range(float x) {
  // (comparisons that leave a NaN a NaN)
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}

__device__ __forceinline__ float f16_bits_to_f32(uint32_t bits, bool bf16) {
  if (bf16) return __uint_as_float(bits << 16);
  union { uint16_t u; _Float16 h; } c;
  c.u = (uint16_t)bits;
  return (float)c.h;
}

// A thread takes 8 values (16 bytes) of a key or value row, or 16 values of a row that is
// stored in 8 bits.  Bytes bound: a row is read once and written once.
template <bool FP8>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppendArgs a, int bf16) {
  const int values = FP8 ? 16 : 8;
  const int pieces = a.D / values, per_token = 2 * a.Hkv * pieces;
  const int64_t first = (int64_t)blockIdx.x * 256 + (threadIdx.x & ~63);
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (first >= (int64_t)a.tokens * per_token) return;
  int seq = 0;
  const int t = (int)(idx / per_token);
  if (a.starts != nullptr) {
    // The sequence of the wavefront's first token, 64 candidates at a time; the other
    // lanes walk on from there.
    const int lane = threadIdx.x & 63, t0 = (int)(first / per_token);
    int lo = 0, hi = a.B;           // the last i in [lo, hi) with starts[i] <= t0
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64;
      const int i = lo + lane * step;
      const uint64_t below = __ballot(i < hi && a.starts[i] <= t0);
      const int n = max(1, (int)__popcll(below));
      hi = min(hi, lo + n * step);
      lo += (n - 1) * step;
    }
    seq = lo;
    if (t < a.tokens)
      while (seq + 1 < a.B && a.starts[seq + 1] <= t) ++seq;
  } else {
    seq = t;
  }
  if (t >= a.tokens || seq >= a.B) return;
  const int rest = (int)(idx - (int64_t)t * per_token);
  const int which = rest / (a.Hkv * pieces), in_row = rest % (a.Hkv * pieces);
  const int h = in_row / pieces, d = (in_row % pieces) * values;
  const int pos = a.starts != nullptr ? a.lens[seq] - a.starts[seq + 1] + t : a.lens[seq] - 1;
  if (pos < 0 || pos >= a.lens[seq]) return;
  const int in_table = pos / a.page_size;
  if (in_table >= a.table_width) return;
  const int page = a.table[(int64_t)seq * a.table_stride + in_table];
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const char* src = (const char*)(which ? a.v : a.k) +
                    ((int64_t)t * (which ? a.v_stride_t : a.k_stride_t) +
                     (int64_t)h * (which ? a.v_stride_h : a.k_stride_h) + d) * 2;
  const int64_t to = (int64_t)page * a.page_stride + (int64_t)h * a.head_stride +
                     (int64_t)(pos - in_table * a.page_size) * a.slot_stride + d;
  char* cache = (char*)(which ? a.v_cache : a.k_cache);
  if constexpr (!FP8) {
    *(u32x4*)(cache + to * 2) = *(const u32x4*)src;
  } else {
    const float scale = (which ? a.v_scale : a.k_scale)[h];
    const u32x4 x[2] = {*(const u32x4*)src, *(const u32x4*)(src + 16)};
    u32x4 codes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = x[i / 2][(i % 2) * 2 + j / 2];
        f[j] = e4m3_range(f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xFFFFu, bf16 != 0) / scale);
      }
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], c, true);
      codes[i] = (uint32_t)c;
    }
    *(u32x4*)(cache + to) = codes;
  }
}

// ---- eviction ----------------------------------------------------------------------------------

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048, kBinCopies = 4;

// A sum as a number that orders as the sums do (NaN above all, -0 like 0).
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive scan over the workgroup of a pair of counts in one word (low and high 16 bits).
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* lds, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(x, d);
    if (lane >= d) x += up;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  *total = all;
  return x + before;
}

// One workgroup for the positions of a sequence in a head.  The least key that is kept is
// found digit by digit (11, 11, 10 bits) from histograms in LDS; then the positions are
// walked in order and the kept ones written down with their sums.
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(const KvEvictArgs a) {
  __shared__ uint32_t bins[kBinCopies][kBins];
  __shared__ uint32_t scan_lds[kSelectWaves];
  __shared__ uint32_t found[2];
  const int t = threadIdx.x, b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const float* const sums = a.sums + (int64_t)b * a.sums_stride_b + (int64_t)h * a.sums_stride_h;
  float* const out = a.sums_out + (int64_t)b * a.out_stride_b + (int64_t)h * a.out_stride_h;
  int32_t* const kept = a.kept + (int64_t)blockIdx.x * a.budget;
  if (h == 0 && t == 0) a.new_lens[b] = min(len, a.budget);
  if (len <= a.budget) {
    for (int j = t; j < a.budget; j += kSelectThreads) kept[j] = j < len ? j : -1;
    if (out != sums)
      for (int j = t; j < len; j += kSelectThreads) out[j] = sums[j];
    return;
  }
  const int lo = a.keep_first, hi = len - a.keep_last;       // positions that have to earn their place
  const int places = a.budget - a.keep_first - a.keep_last;  // (hi - lo > places)
  uint32_t prefix = 0, mask = 0;   // digits of the least key that is kept, so far
  uint32_t need = (uint32_t)places;
  if (places > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, n = pass == 2 ? 1024 : 2048;
      for (int i = t; i < kBinCopies * kBins; i += kSelectThreads) (&bins[0][0])[i] = 0;
      __syncthreads();
      for (int j = lo + t; j < hi; j += kSelectThreads) {
        const uint32_t key = order_key(sums[j]);
        if ((key & mask) == prefix) atomicAdd(&bins[(t >> 6) % kBinCopies][(key >> shift) & (n - 1)], 1u);
      }
      __syncthreads();
      // from the largest digit down: thread t holds the digits n - 1 - 2 t and n - 2 - 2 t
      uint32_t c[2] = {0, 0};
      if (2 * t < n) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < kBinCopies; ++k) c[i] += bins[k][n - 1 - 2 * t - i];
      }
      uint32_t total;
      const uint32_t upto = block_scan(c[0] + c[1], scan_lds, &total);
      uint32_t above = upto - c[0] - c[1];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (c[i] > 0 && above < need && above + c[i] >= need) {
          found[0] = (uint32_t)(n - 1 - 2 * t - i);
          found[1] = need - above;
        }
        above += c[i];
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= (uint32_t)(n - 1) << shift;
      need = found[1];
      __syncthreads();
    }
  }
  // `need`: of the keys equal to the least one, the first so many are kept
  uint32_t n_kept = 0, n_equal = 0;
  for (int j0 = 0; j0 < len; j0 += 4 * kSelectThreads) {
    float x[4];
    uint32_t flags = 0, counts = 0;      // bit i: kept for certain, bit 4 + i: equal to the least key
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + 4 * t + i;
      x[i] = j < len ? sums[j] : 0.0f;
      if (j < len) {
        const uint32_t key = order_key(x[i]);
        if (j < lo || j >= hi || (places > 0 && key > prefix)) {
          flags |= 1u << i;
          counts += 1;
        } else if (places > 0 && key == prefix) {
          flags |= 16u << i;
          counts += 1u << 16;
        }
      }
    }
    uint32_t total;
    const uint32_t upto = block_scan(counts, scan_lds, &total) - counts;
    uint32_t sure = n_kept + (upto & 0xFFFFu), equal = n_equal + (upto >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool is_equal = (flags >> (4 + i)) & 1u;
      if (((flags >> i) & 1u) || (is_equal && equal < need)) {
        // what was kept before it: the certain ones, and of the equal ones at most `need`
        const uint32_t at = sure + min(equal, need);
        kept[at] = j0 + 4 * t + i;
        out[at] = x[i];
      }
      sure += (flags >> i) & 1u;
      equal += is_equal ? 1u : 0u;
    }
    n_kept += total & 0xFFFFu;
    n_equal += total >> 16;
  }
  __syncthreads();
  for (int j = a.budget + t; j < len; j += kSelectThreads) out[j] = 0.0f;
}

// One workgroup for the keys or the values of a sequence in a head: rows move to lower
// places in batches, in order.  Row kept[j] >= j goes to j, so that what a batch writes is
// read by this batch or an earlier one alone: it writes once all its own reads are done.
constexpr int kMoveLoads = 8;
__global__ __launch_bounds__(256) void kv_move_kernel(const KvEvictArgs a) {
  const int which = blockIdx.x & 1, bh = blockIdx.x >> 1, b = bh / a.Hkv, h = bh % a.Hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  if (len <= a.budget) return;
  char* const cache = (char*)(which ? a.v_cache : a.k_cache) + (int64_t)h * a.head_stride;
  const int32_t* const kept = a.kept + (int64_t)bh * a.budget;
  const int32_t* const pages = a.table + (int64_t)b * a.table_stride;
  const int pieces = a.row_bytes / 16;
  const int per_batch = 256 * kMoveLoads;
  const int total = a.budget * pieces;     // (at most 2^31: checked by the entry point)
  for (int e0 = 0; e0 < total; e0 += per_batch) {
    u32x4 x[kMoveLoads];
    char* to[kMoveLoads];
#pragma unroll
    for (int i = 0; i < kMoveLoads; ++i) {
      const int e = e0 + i * 256 + threadIdx.x;
      to[i] = nullptr;
      if (e < total) {
        const int j = e / pieces, piece = e - j * pieces;
        const int src = kept[j];
        if (src != j) {
          const int p0 = j / a.page_size, p1 = src / a.page_size;
          const int page0 = pages[p0], page1 = pages[p1];
          if ((uint32_t)page0 < (uint32_t)a.num_pages && (uint32_t)page1 < (uint32_t)a.num_pages) {
            x[i] = *(const u32x4*)(cache + (int64_t)page1 * a.page_stride +
                                   (int64_t)(src - p1 * a.page_size) * a.slot_stride + piece * 16);
            to[i] = cache + (int64_t)page0 * a.page_stride + (int64_t)(j - p0 * a.page_size) * a.slot_stride + piece * 16;
          }
        }
      }
    }
    // every read of the batch has arrived before any of its rows is written
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoveLoads; ++i)
      if (to[i] != nullptr) *(u32x4*)to[i] = x[i];
  }
}

}  // namespace

void launch_kv_append(const KvAppendArgs& a, int kind, hipStream_t stream) {
  const bool fp8 = kind == kKvFp8Bf16 || kind == kKvFp8F16;
  const int64_t items = (int64_t)a.tokens * 2 * a.Hkv * (a.D / (fp8 ? 16 : 8));
  const dim3 grid((unsigned)((items + 255) / 256)), block(256);
  const int bf16 = kind == kKvBf16 || kind == kKvFp8Bf16;
  if (fp8)
    hipLaunchKernelGGL((kv_append_kernel<true>), grid, block, 0, stream, a, bf16);
  else
    hipLaunchKernelGGL((kv_append_kernel<false>), grid, block, 0, stream, a, bf16);
}

void launch_kv_evict(const KvEvictArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(kv_select_kernel, dim3(a.B * a.Hkv), dim3(kSelectThreads), 0, stream, a);
  hipLaunchKernelGGL(kv_move_kernel, dim3(2 * a.B * a.Hkv), dim3(256), 0, stream, a);
}

}  // namespace vk

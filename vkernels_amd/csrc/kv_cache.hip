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
  const int in_table = divided(pos, a.by_page);
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
constexpr int kSelectLoads = 16;
constexpr int kListed = 512;   // candidates of a wavefront that are kept in LDS

// A sum as a number that orders as the sums do (NaN above all, -0 like 0).
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive sum over the lanes of a wavefront up to this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
#define VK_ADD_FROM(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xF, true)
  VK_ADD_FROM(0x111, 0xF);   // the lane 1, 2, 4, 8 below, within rows of 16
  VK_ADD_FROM(0x112, 0xF);
  VK_ADD_FROM(0x114, 0xF);
  VK_ADD_FROM(0x118, 0xF);
  VK_ADD_FROM(0x142, 0xA);   // lane 15 of rows 0 and 2 to rows 1 and 3
  VK_ADD_FROM(0x143, 0xC);   // lane 31 to rows 2 and 3
#undef VK_ADD_FROM
  return x;
}

// Of the digits counted in `bins` (n of them): the one that the need-th largest key has,
// found[0], and how many keys of it are still wanted, found[1].
__device__ void find_digit(uint32_t (*bins)[kBins], int n, uint32_t need, uint32_t* scan_lds, uint32_t* found) {
  const int t = threadIdx.x, wave = t >> 6;
  // from the largest digit down: thread t holds the digits n - 1 - 2 t and n - 2 - 2 t
  uint32_t c[2] = {0, 0};
  if (2 * t < n) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < kBinCopies; ++k) c[i] += bins[k][n - 1 - 2 * t - i];
  }
  uint32_t above = wave_scan(c[0] + c[1]);
  if ((t & 63) == 63) scan_lds[wave] = above;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w)
    if (w < wave) above += scan_lds[w];
  above -= c[0] + c[1];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (c[i] > 0 && above < need && above + c[i] >= need) {
      found[0] = (uint32_t)(n - 1 - 2 * t - i);
      found[1] = need - above;
    }
    above += c[i];
  }
  __syncthreads();
}

// One workgroup for the positions of a sequence in a head.  The least key that is kept is
// found digit by digit (11, 11, 10 bits) from histograms in LDS.  The first pass reads the
// sums; the second, when the first digit is known, counts what is kept for certain and
// lists the keys that share the digit in LDS, where the other two digits are found (the
// sums are read again for those when there are too many such keys).  The last pass writes
// the kept positions down: every wavefront walks a stretch of its own, from the counts of
// the ones before it.
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(const KvEvictArgs a) {
  __shared__ uint32_t bins[kBinCopies][kBins];
  __shared__ uint32_t listed[kSelectWaves][kListed];
  __shared__ uint32_t scan_lds[kSelectWaves], sure_of[kSelectWaves], equal_of[kSelectWaves];
  __shared__ uint32_t found[2], too_many;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
  // What orders the workgroups of the compaction behind this, for the keys and the values: a
  // count of the batches taken, and a word for each batch that has been read.
  for (int i = t; i < 2 * (1 + a.batches); i += kSelectThreads)
    a.order[(int64_t)blockIdx.x * 2 * (1 + a.batches) + i] = 0;

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
  const uint32_t places = (uint32_t)(a.budget - a.keep_first - a.keep_last);   // (hi - lo > places)
  const int stretch = (len + 64 * kSelectWaves - 1) / (64 * kSelectWaves) * 64;
  const int from = min(len, wave * stretch), to = min(len, from + stretch);
  // The sums of 1024 positions of the stretch at a time, 16 a lane: all their loads at once, and
  // none but the first pass's where that is the whole stretch (up to 16384 positions).
  float x[kSelectLoads];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kSelectLoads; ++i) {
      const int j = j0 + 64 * i + lane;
      if (j0 + 64 * i < to) x[i] = sums[min(j, to - 1)];
    }
  };
  const bool resident = stretch <= 64 * kSelectLoads;
  // f(position, is it one, sum) for every position of the stretch, in order; `again`: a pass
  // behind the first.
  auto walk = [&](bool again, auto f) {
    for (int j0 = from; j0 < to; j0 += 64 * kSelectLoads) {
      if (!again || !resident) load(j0);
#pragma unroll
      for (int i = 0; i < kSelectLoads; ++i)
        if (j0 + 64 * i < to) f(j0 + 64 * i + lane, j0 + 64 * i + lane < to, x[i]);
    }
  };

  uint32_t least = 0, need = places;   // the least key that is kept; of its equals, the first `need` are
  auto clear_bins = [&] {
    for (int i = t; i < kBinCopies * kBins; i += kSelectThreads) (&bins[0][0])[i] = 0;
    __syncthreads();
  };
  clear_bins();
  walk(false, [&](int j, bool real, float v) {
    if (real && j >= lo && j < hi) atomicAdd(&bins[wave % kBinCopies][order_key(v) >> 21], 1u);
  });
  if (t == 0) too_many = 0;
  __syncthreads();
  if (places > 0) {
    find_digit(bins, 2048, places, scan_lds, found);
    least = found[0] << 21;
    need = found[1];
  }

  // what this wavefront's stretch keeps for certain, and its candidates
  uint32_t sure = 0, n_listed = 0;
  const uint64_t below = (1ull << lane) - 1;
  walk(true, [&](int j, bool real, float v) {
    const uint32_t key = order_key(v);
    const bool ends = real && (j < lo || j >= hi), middle = real && !ends && places > 0;
    sure += (uint32_t)__popcll(__ballot(ends || (middle && key >> 21 > least >> 21)));
    const bool candidate = middle && key >> 21 == least >> 21;
    const uint64_t all = __ballot(candidate);
    const uint32_t at = n_listed + (uint32_t)__popcll(all & below);
    if (candidate && at < kListed) listed[wave][at] = key;
    n_listed += (uint32_t)__popcll(all);
  });
  uint32_t equal = 0;
  if (places > 0) {
    if (lane == 0 && n_listed > kListed) too_many = 1;
    __syncthreads();
    const bool again = too_many != 0;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      const int shift = pass == 0 ? 10 : 0, n = pass == 0 ? 2048 : 1024;
      const uint32_t same = pass == 0 ? 21 : 10;    // the bits above agree
      clear_bins();
      if (!again) {
        for (uint32_t i = lane; i < n_listed; i += 64) {
          const uint32_t key = listed[wave][i];
          if (key >> same == least >> same) atomicAdd(&bins[wave % kBinCopies][(key >> shift) & (n - 1)], 1u);
        }
      } else {
        walk(true, [&](int j, bool real, float v) {
          const uint32_t key = order_key(v);
          if (real && j >= lo && j < hi && key >> same == least >> same)
            atomicAdd(&bins[wave % kBinCopies][(key >> shift) & (n - 1)], 1u);
        });
      }
      __syncthreads();
      find_digit(bins, n, need, scan_lds, found);
      least |= found[0] << shift;
      need = found[1];
      __syncthreads();
    }
    if (!again) {
      for (uint32_t i0 = 0; i0 < n_listed; i0 += 64) {
        const bool real = i0 + lane < n_listed;
        const uint32_t key = real ? listed[wave][i0 + lane] : 0u;
        sure += (uint32_t)__popcll(__ballot(real && key > least));
        equal += (uint32_t)__popcll(__ballot(real && key == least));
      }
    } else {
      walk(true, [&](int j, bool real, float v) {
        const bool middle = real && j >= lo && j < hi;
        const uint32_t key = order_key(v);
        sure += (uint32_t)__popcll(__ballot(middle && key > least && key >> 21 == least >> 21));
        equal += (uint32_t)__popcll(__ballot(middle && key == least));
      });
    }
  }
  if (lane == 0) {
    sure_of[wave] = sure;
    equal_of[wave] = equal;
  }
  __syncthreads();
  uint32_t n_sure = 0, n_equal = 0;     // kept before this wavefront's stretch
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    if (w < wave) {
      n_sure += sure_of[w];
      n_equal += equal_of[w];
    }
  }
  const bool in_place = out == sums;
  walk(true, [&](int j, bool real, float v) {
    const uint32_t key = order_key(v);
    const bool ends = real && (j < lo || j >= hi), middle = real && !ends && places > 0;
    const bool certain = ends || (middle && key > least), tied = middle && key == least;
    const uint64_t certain_all = __ballot(certain), tied_all = __ballot(tied);
    const uint32_t ties = n_equal + (uint32_t)__popcll(tied_all & below);
    if (certain || (tied && ties < need)) {
      // what was kept before it: the certain ones, and of the equal ones at most `need`
      const uint32_t at = n_sure + (uint32_t)__popcll(certain_all & below) + min(ties, need);
      kept[at] = j;
      if (!in_place) out[at] = v;
    }
    n_sure += (uint32_t)__popcll(certain_all);
    n_equal += (uint32_t)__popcll(tied_all);
  });
  __syncthreads();
  if (in_place) {
    // kept[j] >= j: a chunk's sums are all read before any of them is written
    for (int j0 = 0; j0 < a.budget; j0 += kSelectThreads) {
      const int j = j0 + t;
      float x = 0.0f;
      if (j < a.budget) x = sums[kept[j]];
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (j < a.budget) out[j] = x;
    }
    __syncthreads();
  }
  for (int j = a.budget + t; j < len; j += kSelectThreads) out[j] = 0.0f;
}

// The compaction.  A batch is 32 KB of rows that become neighbours: the keys or the values
// of a head, kept[j] -> j for `rows` successive j.  A workgroup reads its batch into
// registers, says so, and writes once every batch that reads what it overwrites has been
// read.  kept[j] >= j grows with j, so those are earlier batches of the same list; the
// workgroups of a list take its batches in the order in which they start, and say that
// they have read without waiting for anything: every wait ends.
constexpr int kMoveLoads = 8, kMoveThreads = 256;
constexpr int kMovePieces = kMoveLoads * kMoveThreads;    // of 16 bytes
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(const KvEvictArgs a) {
  __shared__ uint32_t ticket_lds;
  const int t = threadIdx.x;
  const int list = blockIdx.x % (2 * a.B * a.Hkv);
  const int which = list & 1, bh = list >> 1, b = bh / a.Hkv, h = bh % a.Hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  if (len <= a.budget) return;
  uint32_t* const taken = a.order + (int64_t)list * (1 + a.batches);
  uint32_t* const read = taken + 1;
  if (t == 0) ticket_lds = __hip_atomic_fetch_add(taken, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const int batch = (int)ticket_lds;
  char* const cache = (char*)(which ? a.v_cache : a.k_cache) + (int64_t)h * a.head_stride;
  const int32_t* const kept = a.kept + (int64_t)bh * a.budget;
  const int32_t* const pages = a.table + (int64_t)b * a.table_stride;
  const int pieces = a.row_bytes / 16, rows = kMovePieces / pieces;
  const int first = batch * rows, last = min(a.budget, first + rows);     // rows that are written
  // Three rounds of loads, each of them all at once: the old places, the pages, the rows.  (A lane
  // without a row, or with one that stays, reads a valid one and writes nothing.)
  int dst[kMoveLoads], src[kMoveLoads], piece[kMoveLoads];
  int dst_page[kMoveLoads], src_page[kMoveLoads];
  bool moves[kMoveLoads];
#pragma unroll
  for (int i = 0; i < kMoveLoads; ++i) {
    const int e = i * kMoveThreads + t, in_batch = divided(e, a.by_pieces);
    piece[i] = e - in_batch * pieces;
    dst[i] = min(first + in_batch, last - 1);
    moves[i] = in_batch < rows && first + in_batch < last;
    src[i] = kept[dst[i]];
  }
#pragma unroll
  for (int i = 0; i < kMoveLoads; ++i) {
    moves[i] = moves[i] && src[i] != dst[i];
    dst_page[i] = pages[divided(dst[i], a.by_page)];
    src_page[i] = pages[divided(src[i], a.by_page)];
  }
  u32x4 x[kMoveLoads];
#pragma unroll
  for (int i = 0; i < kMoveLoads; ++i) {
    const bool there = (uint32_t)src_page[i] < (uint32_t)a.num_pages;
    moves[i] = moves[i] && there && (uint32_t)dst_page[i] < (uint32_t)a.num_pages;
    const int slot = src[i] - divided(src[i], a.by_page) * a.page_size;
    x[i] = *(const u32x4*)(cache + (there ? (int64_t)src_page[i] * a.page_stride + (int64_t)slot * a.slot_stride : 0) +
                           piece[i] * 16);
  }
  // Every read of the batch has arrived: the rows are in registers, and nobody reads in this
  // kernel what another workgroup writes, so that the words need no cache to be written
  // back or invalidated (relaxed, but seen by the whole card).
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (t == 0) __hip_atomic_store(read + batch, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // earlier batches with a source among the rows first .. last - 1
  for (int c = t; c < batch; c += kMoveThreads) {
    if (kept[c * rows] < last && kept[c * rows + rows - 1] >= first)
      while (__hip_atomic_load(read + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) __builtin_amdgcn_s_sleep(2);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMoveLoads; ++i) {
    const int slot = dst[i] - divided(dst[i], a.by_page) * a.page_size;
    if (moves[i])
      *(u32x4*)(cache + (int64_t)dst_page[i] * a.page_stride + (int64_t)slot * a.slot_stride + piece[i] * 16) = x[i];
  }
}

}  // namespace

void launch_kv_append(const KvAppendArgs& args, int kind, hipStream_t stream) {
  KvAppendArgs a = args;
  a.by_page = fast_div(a.page_size);
  const bool fp8 = kind == kKvFp8Bf16 || kind == kKvFp8F16;
  const int64_t items = (int64_t)a.tokens * 2 * a.Hkv * (a.D / (fp8 ? 16 : 8));
  const dim3 grid((unsigned)((items + 255) / 256)), block(256);
  const int bf16 = kind == kKvBf16 || kind == kKvFp8Bf16;
  if (fp8)
    hipLaunchKernelGGL((kv_append_kernel<true>), grid, block, 0, stream, a, bf16);
  else
    hipLaunchKernelGGL((kv_append_kernel<false>), grid, block, 0, stream, a, bf16);
}

int kv_evict_batches(int budget, int row_bytes) {
  const int rows = kMovePieces / (row_bytes / 16);
  return (budget + rows - 1) / rows;
}

void launch_kv_evict(const KvEvictArgs& args, hipStream_t stream) {
  KvEvictArgs a = args;
  a.by_page = fast_div(a.page_size);
  a.by_pieces = fast_div(a.row_bytes / 16);
  hipLaunchKernelGGL(kv_select_kernel, dim3(a.B * a.Hkv), dim3(kSelectThreads), 0, stream, a);
  hipLaunchKernelGGL(kv_move_kernel, dim3(2 * a.B * a.Hkv * a.batches), dim3(kMoveThreads), 0, stream, a);
}

}  // namespace vk

// kv_cache.hip — new rows into a paged key-value cache, and its eviction by accumulated
// attention weight: the positions of most weight are selected and the cache is compacted
// to them, in place.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv_cache.hpp"
#include "paged_attention.hpp"

namespace vk {
namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

// ---- append --------------------------------------------------------------------------------

// What does not fit into E4M3 is stored as its largest finite code.
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

// 8 values of a row as E4M3 codes.
__device__ __forceinline__ u32x2 e4m3_codes(u32x4 x, float scale, bool bf16) {
  u32x2 codes;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = x[2 * i + j / 2];
      f[j] = e4m3_range(f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xFFFFu, bf16) / scale);
    }
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], c, true);
    codes[i] = (uint32_t)c;
  }
  return codes;
}

// A thread takes the same 8 values (16 bytes) of a token's key and value in a head.  The rows are
// asked for before their place is looked up: length, then page, then store are the latency that
// a decode step's call consists of (4 us for 255 tokens); a prompt's is bound by the rows read
// and written (8191 tokens of 8 heads of 128: 67 MB in 13.9 us, 4.8 TB/s; a thread for each key
// or value, its row behind the look-up, took 17).  Into an 8-bit cache these tokens take 15.7 us (50 MB):
// 16 IEEE divisions a thread, and stores of half the width.
template <bool FP8>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppendArgs a, int bf16) {
  const int per_token = a.Hkv * a.pieces;
  const int first = (int)(blockIdx.x * 256 + (threadIdx.x & ~63)), idx = (int)(blockIdx.x * 256 + threadIdx.x);
  if (first >= a.tokens * per_token) return;
  const int t = divided(idx, a.by_token), rest = idx - t * per_token;
  const int h = divided(rest, a.by_pieces), d = (rest - h * a.pieces) * 8;
  const int there = min(t, a.tokens - 1);
  const u32x4 k = *(const u32x4*)((const char*)a.k + ((int64_t)there * a.k_stride_t + (int64_t)h * a.k_stride_h + d) * 2);
  const u32x4 v = *(const u32x4*)((const char*)a.v + ((int64_t)there * a.v_stride_t + (int64_t)h * a.v_stride_h + d) * 2);
  int seq = there;
  if (a.starts != nullptr) {
    // The sequence of the wavefront's first token, 64 candidates at a time; the other
    // lanes walk on from there.
    const int lane = threadIdx.x & 63, t0 = divided(first, a.by_token);
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
    while (seq + 1 < a.B && a.starts[seq + 1] <= there) ++seq;
  }
  if (t >= a.tokens || seq >= a.B || (a.starts != nullptr && t < a.starts[seq])) return;
  const int len = a.lens[seq];
  const int pos = a.starts != nullptr ? len - a.starts[seq + 1] + t : len - 1;
  if (pos < 0 || pos >= len) return;
  const int in_table = divided(pos, a.by_page);
  if (in_table >= a.table_width) return;
  const int page = a.table[(int64_t)seq * a.table_stride + in_table];
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int64_t to = (int64_t)page * a.page_stride + (int64_t)h * a.head_stride +
                     (int64_t)(pos - in_table * a.page_size) * a.slot_stride + d;
  if constexpr (!FP8) {
    *(u32x4*)((char*)a.k_cache + to * 2) = k;
    *(u32x4*)((char*)a.v_cache + to * 2) = v;
  } else {
    *(u32x2*)((char*)a.k_cache + to) = e4m3_codes(k, a.k_scale[h], bf16 != 0);
    *(u32x2*)((char*)a.v_cache + to) = e4m3_codes(v, a.v_scale[h], bf16 != 0);
  }
}

// ---- eviction ----------------------------------------------------------------------------------

// A row's workgroup: 16 wavefronts, or 4 for short and for many rows.  (The split form: 16.)
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64, kFewThreads = 256;
constexpr int kBins = 2048;
constexpr int bin_copies(int threads) { return threads / 256; }
constexpr int kSelectLoads = 8;
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

// The workgroup's threads hold the counts c of N successive digits each, from the largest digit
// down (thread t those of digits n - 1 - N t and below).  Finds the digit that the need-th
// largest key has, found[0], and how many keys of it are still wanted, found[1].
template <int THREADS, int N>
__device__ void find_digit(const uint32_t (&c)[N], int n, uint32_t need, uint32_t* scan_lds, uint32_t* found) {
  static_assert(N * THREADS == kBins, "a thread for every N digits");
  const int t = threadIdx.x, wave = t >> 6;
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) mine += c[i];
  uint32_t above = wave_scan(mine);
  if ((t & 63) == 63) scan_lds[wave] = above;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w)
    if (w < wave) above += scan_lds[w];
  above -= mine;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (c[i] > 0 && above < need && above + c[i] >= need) {
      found[0] = (uint32_t)(n - 1 - N * t - i);
      found[1] = need - above;
    }
    above += c[i];
  }
  __syncthreads();
}

// The same from histograms in LDS.
template <int THREADS>
__device__ void find_digit_lds(uint32_t (*bins)[kBins], int n, uint32_t need, uint32_t* scan_lds, uint32_t* found) {
  constexpr int N = kBins / THREADS;
  uint32_t c[N] = {};
  if (N * (int)threadIdx.x < n) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < bin_copies(THREADS); ++k) c[i] += bins[k][n - 1 - N * threadIdx.x - i];
  }
  find_digit<THREADS>(c, n, need, scan_lds, found);
}

// The digits, from the most significant one: their shifts, numbers of values and the bits above.
__device__ __forceinline__ constexpr int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ constexpr int digit_values(int pass) { return pass == 2 ? 1024 : 2048; }

// A row of sums (a sequence in a head) that is cut, and the stretch of it that a wavefront
// walks.
struct SelectRow {
  int len, lo, hi;      // positions; those in [lo, hi) have to earn their place
  uint32_t places;      // how many of them do (fewer than there are, those without a page not counted)
  const int32_t* pages;
  int num_pages;
  FastDiv by_page;
  const float* sums;
  int32_t* kept;
  int from, to;         // the wavefront's stretch
  int lane;
  bool resident;        // the stretch is held in registers after the first pass

  // f(position, is it one, sum) for every position of the stretch, in order, 64 at a time; the sums
  // of 64 kSelectLoads positions are loaded at once, and only by the first pass (`again` false)
  // where that is the whole stretch.
  template <class F>
  __device__ __forceinline__ void walk(float (&x)[kSelectLoads], bool again, F f) const {
    for (int j0 = from; j0 < to; j0 += 64 * kSelectLoads) {
      if (!again || !resident) load(x, j0);
#pragma unroll
      for (int i = 0; i < kSelectLoads; ++i)
        if (j0 + 64 * i < to) f(j0 + 64 * i + lane, j0 + 64 * i + lane < to, x[i]);
    }
  }
  __device__ __forceinline__ void load(float (&x)[kSelectLoads], int j0) const {
#pragma unroll
    for (int i = 0; i < kSelectLoads; ++i)
      if (j0 + 64 * i < to) x[i] = sums[min(j0 + 64 * i + lane, to - 1)];
  }
  // (ahead of other work, so that the first pass finds the sums there: it is then one `again`)
  __device__ __forceinline__ void preload(float (&x)[kSelectLoads]) const {
    if (resident) load(x, from);
  }
  __device__ __forceinline__ bool has_page(int j) const {
    return (uint32_t)pages[divided(j, by_page)] < (uint32_t)num_pages;
  }
  // (HOLES: there are positions without a page, which are never kept.  Rows that have none, all but a few, take
  // code of their own, without the look-ups in each pass.)
  template <bool HOLES>
  __device__ __forceinline__ bool earns(int j, bool real) const {
    return real && j >= lo && j < hi && (!HOLES || has_page(j));
  }
  __device__ __forceinline__ bool given(int j, bool real) const { return real && (j < lo || j >= hi); }
};

// Row and stretch of `part` of `parts` workgroups of a row, a stretch for each of their wavefronts; whether
// it is longer than the budget.
template <int THREADS>
__device__ __forceinline__ bool select_row(const KvEvictArgs& a, int row, int part, int parts, SelectRow* r) {
  const int t = threadIdx.x, wave = t >> 6, b = row / a.Hkv, h = row % a.Hkv;
  r->len = min(max(a.lens[b], 0), a.max_len);
  r->sums = a.sums + (int64_t)b * a.sums_stride_b + (int64_t)h * a.sums_stride_h;
  r->kept = a.kept + (int64_t)row * a.budget;
  r->pages = a.table + (int64_t)b * a.table_stride;
  r->num_pages = a.num_pages;
  r->by_page = a.by_page;
  r->lane = t & 63;
  r->lo = a.keep_first;
  r->hi = r->len - a.keep_last;
  r->places = (uint32_t)(a.budget - a.keep_first - a.keep_last);
  const int waves = parts * (THREADS / 64);
  const int stretch = (r->len + 64 * waves - 1) / (64 * waves) * 64;
  r->from = min(r->len, (part * (THREADS / 64) + wave) * stretch);
  r->to = min(r->len, r->from + stretch);
  r->resident = stretch <= 64 * kSelectLoads;
  return r->len > a.budget;
}

// Positions [from, to) of the row without a page, as a wavefront finds them: are there any, and is one of them
// the new place of a kept position or kept itself (such a row is not cut).  Each wavefront looks through the
// pages of its stretch: 1 us of the 15 that 512 rows of 2304 sums take, 0.7 of 27 for 6976 rows of up to 64.
constexpr uint32_t kHole = 1, kHoleInTheWay = 2;
__device__ __forceinline__ uint32_t find_holes(const KvEvictArgs& a, const SelectRow& r, int from, int to) {
  const int last = to > from ? divided(to - 1, r.by_page) : -1;
  uint32_t mine = 0;
#pragma unroll 4
  for (int i = divided(from, r.by_page) + r.lane; i <= last; i += 64) {
    if ((uint32_t)r.pages[i] >= (uint32_t)r.num_pages) {
      const int first = i * a.page_size, behind = (int)min((int64_t)first + a.page_size, (int64_t)r.len);
      mine |= first < a.budget || behind > r.hi ? kHole | kHoleInTheWay : kHole;
    }
  }
  return (__any(mine & kHole) ? kHole : 0u) | (__any(mine & kHoleInTheWay) ? kHoleInTheWay : 0u);
}
// The wavefronts' findings, left in LDS in front of a barrier.
template <int WAVES>
__device__ __forceinline__ uint32_t all_holes(const uint32_t* holes_lds) {
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) all |= holes_lds[w];
  return __builtin_amdgcn_readfirstlane(all);
}

// What the first launch leaves for the compaction besides the kept positions: the new length of a row that
// is cut, and the order of its workgroups (for the keys and the values a count of the batches taken, and a
// word for each batch that has been read).
template <int THREADS>
__device__ __forceinline__ void open_row(const KvEvictArgs& a, int row, const SelectRow& r) {
  const int t = threadIdx.x, b = row / a.Hkv, h = row % a.Hkv;
  for (int i = t; i < 2 * (1 + a.batches); i += THREADS) a.order[(int64_t)row * 2 * (1 + a.batches) + i] = 0;
  if (h == 0 && t == 0) a.new_lens[b] = min(r.len, a.budget);
}
// All there is of a row that is not cut.
template <int THREADS>
__device__ void leave_row(const KvEvictArgs& a, int row, const SelectRow& r) {
  const int t = threadIdx.x, b = row / a.Hkv, h = row % a.Hkv;
  if (h == 0 && t == 0) a.new_lens[b] = r.len;
  float* const out = a.sums_out + (int64_t)b * a.out_stride_b + (int64_t)h * a.out_stride_h;
  for (int j = t; j < a.budget; j += THREADS) r.kept[j] = j < r.len ? j : -1;
  if (out != r.sums)
    for (int j = t; j < r.len; j += THREADS) out[j] = r.sums[j];
}

// The last pass: the wavefront's kept positions, behind the `certain` and `ties` ones before its stretch;
// of the keys equal to `least` the first `need` of the row are kept.
template <bool HOLES>
__device__ __forceinline__ void write_kept(const SelectRow& r, float (&x)[kSelectLoads], uint32_t least, uint32_t need,
                                           uint32_t certain, uint32_t ties) {
  const uint64_t below = (1ull << r.lane) - 1;
  r.walk(x, true, [&](int j, bool real, float v) {
    const uint32_t key = order_key(v);
    const bool middle = r.earns<HOLES>(j, real) && r.places > 0;
    const bool sure = r.given(j, real) || (middle && key > least), tied = middle && key == least;
    const uint64_t all_sure = __ballot(sure), all_tied = __ballot(tied);
    const uint32_t before = ties + (uint32_t)__popcll(all_tied & below);
    // what was kept before it: the certain ones, and of the equal ones at most `need`
    if (sure || (tied && before < need))
      r.kept[certain + (uint32_t)__popcll(all_sure & below) + min(before, need)] = j;
    certain += (uint32_t)__popcll(all_sure);
    ties += (uint32_t)__popcll(all_tied);
  });
}

// Sums over the workgroup's wavefronts before this one, of a pair of counts.
template <int WAVES>
__device__ __forceinline__ void counts_before(uint32_t& sure, uint32_t& equal, uint32_t (*lds)[WAVES]) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    lds[0][wave] = sure;
    lds[1][wave] = equal;
  }
  __syncthreads();
  sure = equal = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) {
      sure += lds[0][w];
      equal += lds[1][w];
    }
  }
}

// One workgroup for a row.  The least key that is kept is found digit by digit (11, 11, 10
// bits) from histograms in LDS.  The first pass reads the sums; the second, when the first
// digit is known, counts what is kept for certain and lists the keys that share the digit in
// LDS, where the other two digits are found (the sums are walked again for those when there
// are too many such keys).  The last pass writes the kept positions down: every wavefront
// walks a stretch of its own, from the counts of the ones before it.
// Bound by its barriers and dependent loads: 512 rows of 2304 sums (9 MB in and out) in 15 us (21
// with 16 sums a lane in registers, which leave a CU room for one workgroup); 32 rows of 65536 in 58 us,
// a CU each, where the split form takes 32.
// (Pointers to arrays of their own: as members of one struct in LDS these cost 9 us for 6976 rows of up to 64
// positions.)
template <int THREADS>
struct SelectLds {
  uint32_t (*bins)[kBins];
  uint32_t (*listed)[kListed];
  uint32_t *scan, (*counts)[THREADS / 64], *found, *too_many;
};

template <int THREADS, bool HOLES>
__device__ void select_kept(const SelectRow& r, float (&x)[kSelectLoads], const SelectLds<THREADS> lds) {
  constexpr int kBinCopies = bin_copies(THREADS);
  const int t = threadIdx.x, wave = t >> 6;
  uint32_t least = 0, need = r.places;   // the least key that is kept; of its equals, the first `need` are
  auto clear_bins = [&] {
    for (int i = t; i < kBinCopies * kBins; i += THREADS) (&lds.bins[0][0])[i] = 0;
    __syncthreads();
  };
  auto count = [&](uint32_t digit) { atomicAdd(&lds.bins[wave % kBinCopies][digit], 1u); };
  r.walk(x, false, [&](int j, bool real, float v) {
    if (r.template earns<HOLES>(j, real)) count(order_key(v) >> 21);
  });
  if (t == 0) *lds.too_many = 0;
  __syncthreads();
  if (r.places > 0) {
    find_digit_lds<THREADS>(lds.bins, 2048, r.places, lds.scan, lds.found);
    least = lds.found[0] << 21;
    need = lds.found[1];
  }

  // what this wavefront's stretch keeps for certain, and its candidates
  uint32_t sure = 0, equal = 0, n_listed = 0;
  const uint64_t below = (1ull << r.lane) - 1;
  r.walk(x, true, [&](int j, bool real, float v) {
    const uint32_t key = order_key(v);
    const bool middle = r.template earns<HOLES>(j, real) && r.places > 0;
    sure += (uint32_t)__popcll(__ballot(r.given(j, real) || (middle && key >> 21 > least >> 21)));
    const bool candidate = middle && key >> 21 == least >> 21;
    const uint64_t all = __ballot(candidate);
    const uint32_t at = n_listed + (uint32_t)__popcll(all & below);
    if (candidate && at < kListed) lds.listed[wave][at] = key;
    n_listed += (uint32_t)__popcll(all);
  });
  if (r.places > 0) {
    if (r.lane == 0 && n_listed > kListed) *lds.too_many = 1;
    __syncthreads();
    const bool again = *lds.too_many != 0;
#pragma unroll 1
    for (int pass = 1; pass < 3; ++pass) {
      const int shift = digit_shift(pass), n = digit_values(pass);
      const uint32_t same = pass == 1 ? 21 : 10;    // the bits above agree
      clear_bins();
      if (!again) {
        for (uint32_t i = r.lane; i < n_listed; i += 64) {
          const uint32_t key = lds.listed[wave][i];
          if (key >> same == least >> same) count((key >> shift) & (n - 1));
        }
      } else {
        r.walk(x, true, [&](int j, bool real, float v) {
          const uint32_t key = order_key(v);
          if (r.template earns<HOLES>(j, real) && key >> same == least >> same) count((key >> shift) & (n - 1));
        });
      }
      __syncthreads();
      find_digit_lds<THREADS>(lds.bins, n, need, lds.scan, lds.found);
      least |= lds.found[0] << shift;
      need = lds.found[1];
      __syncthreads();
    }
    if (!again) {
      for (uint32_t i0 = 0; i0 < n_listed; i0 += 64) {
        const bool real = i0 + r.lane < n_listed;
        const uint32_t key = real ? lds.listed[wave][i0 + r.lane] : 0u;
        sure += (uint32_t)__popcll(__ballot(real && key > least));
        equal += (uint32_t)__popcll(__ballot(real && key == least));
      }
    } else {
      r.walk(x, true, [&](int j, bool real, float v) {
        const bool middle = r.template earns<HOLES>(j, real);
        const uint32_t key = order_key(v);
        sure += (uint32_t)__popcll(__ballot(middle && key > least && key >> 21 == least >> 21));
        equal += (uint32_t)__popcll(__ballot(middle && key == least));
      });
    }
  }
  counts_before(sure, equal, lds.counts);
  write_kept<HOLES>(r, x, least, need, sure, equal);
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(const KvEvictArgs a) {
  __shared__ uint32_t bins[bin_copies(THREADS)][kBins];
  __shared__ uint32_t listed[THREADS / 64][kListed];
  __shared__ uint32_t scan_lds[THREADS / 64], counts_lds[2][THREADS / 64], holes_lds[THREADS / 64];
  __shared__ uint32_t found[2], too_many;
  const SelectLds<THREADS> lds = {bins, listed, scan_lds, counts_lds, found, &too_many};
  const int t = threadIdx.x, wave = t >> 6;
  SelectRow r;
  const bool longer = select_row<THREADS>(a, blockIdx.x, 0, 1, &r);
  open_row<THREADS>(a, blockIdx.x, r);
  if (!longer) {
    leave_row<THREADS>(a, blockIdx.x, r);
    return;
  }
  float x[kSelectLoads];
  const uint32_t mine = find_holes(a, r, r.from, r.to);
  if (r.lane == 0) holes_lds[wave] = mine;
  for (int i = t; i < bin_copies(THREADS) * kBins; i += THREADS) (&bins[0][0])[i] = 0;
  __syncthreads();
  const uint32_t holes = all_holes<THREADS / 64>(holes_lds);
  if (holes == 0)
    select_kept<THREADS, false>(r, x, lds);
  else if (holes & kHoleInTheWay)
    leave_row<THREADS>(a, blockIdx.x, r);
  else
    select_kept<THREADS, true>(r, x, lds);
}

// Few long rows: `parts` workgroups for each, a launch for each digit.  A workgroup counts the
// digits of its part and leaves the counts in the workspace; the next launch adds the parts' counts
// up and goes on from the digit found.  What a part keeps for certain follows from the counts as
// well, so that the last launch knows where each part's positions begin.
constexpr int kMostParts = 16;
// (even: pairs of counts are read)
__host__ __device__ constexpr int kv_split_words(int parts) { return 3 * parts * kBins + 4 + 3 * parts + (parts & 1); }
struct SplitRow {
  uint32_t* counts;   // [3][parts][kBins]
  uint32_t* state;    // least, need behind digit 0 and behind digit 1; [2][parts] kept before a part by those;
                      // [parts] the parts' positions without a page
};
__device__ __forceinline__ SplitRow split_row(const KvEvictArgs& a, int row) {
  const int words = kv_split_words(a.parts);
  uint32_t* const base = a.split + (int64_t)row * words;
  return SplitRow{base, base + 3 * a.parts * kBins};
}

// Digit `pass` of the least key from the parts' counts, and of the keys in the parts before this one
// how many are above it by this digit, and how many share it.  Part 0 leaves what is known
// behind digits 0 and 1, every part its own count above by them.
struct PartsBefore {
  uint32_t above, equal;
};
__device__ PartsBefore split_digit(const KvEvictArgs& a, const SplitRow& s, int pass, int part, uint32_t& least,
                                   uint32_t& need, uint32_t (*lds)[kSelectWaves], uint32_t* found) {
  const int t = threadIdx.x, n = digit_values(pass);
  uint32_t c[2] = {0, 0}, before[2] = {0, 0};
  if (2 * t < n) {
    const uint32_t* const from = s.counts + (int64_t)pass * a.parts * kBins + (n - 2 - 2 * t);
    uint64_t pair[kMostParts];      // both digits of a part, all parts' loads at once
#pragma unroll
    for (int p = 0; p < kMostParts; ++p) pair[p] = p < a.parts ? *(const uint64_t*)(from + p * kBins) : 0ull;
#pragma unroll
    for (int p = 0; p < kMostParts; ++p) {
      const uint32_t high = (uint32_t)(pair[p] >> 32), low = (uint32_t)pair[p];
      c[0] += high;
      c[1] += low;
      before[0] += p < part ? high : 0u;
      before[1] += p < part ? low : 0u;
    }
  }
  find_digit<kSelectThreads>(c, n, need, lds[0], found);
  const uint32_t digit = found[0];
  least |= digit << digit_shift(pass);
  need = found[1];
  uint32_t above = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t mine = (uint32_t)(n - 1 - 2 * t - i);
    if (2 * t < n) {
      above += mine > digit ? before[i] : 0u;
      equal += mine == digit ? before[i] : 0u;
    }
  }
  above = wave_scan(above);
  equal = wave_scan(equal);
  if ((t & 63) == 63) {
    lds[0][t >> 6] = above;
    lds[1][t >> 6] = equal;
  }
  __syncthreads();
  PartsBefore r = {0, 0};
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    r.above += lds[0][w];
    r.equal += lds[1][w];
  }
  if (t == 0 && pass < 2) {
    s.state[4 + pass * a.parts + part] = r.above;
    if (part == 0) {
      s.state[2 * pass] = least;
      s.state[2 * pass + 1] = need;
    }
  }
  return r;
}

// All parts' positions without a page, behind the first launch.
__device__ __forceinline__ uint32_t split_holes(const KvEvictArgs& a, const SplitRow& s) {
  uint32_t all = 0;
#pragma unroll
  for (int p = 0; p < kMostParts; ++p) all |= p < a.parts ? s.state[4 + 2 * a.parts + p] : 0u;
  return __builtin_amdgcn_readfirstlane(all);
}

// The digits of the part's keys that agree with `least` so far.
template <int PASS, bool HOLES>
__device__ __forceinline__ void count_digits(const SelectRow& r, float (&x)[kSelectLoads], uint32_t least, uint32_t* bins) {
  r.walk(x, true, [&](int j, bool real, float v) {
    const uint32_t key = order_key(v);
    constexpr uint32_t same = PASS == 1 ? 21 : 10;
    if (r.template earns<HOLES>(j, real) && (PASS == 0 || key >> same == least >> same))
      atomicAdd(bins + ((key >> digit_shift(PASS)) & (digit_values(PASS) - 1)), 1u);
  });
}

template <int PASS>
__global__ __launch_bounds__(kSelectThreads) void kv_select_digit_kernel(const KvEvictArgs a) {
  constexpr int kBinCopies = bin_copies(kSelectThreads);
  __shared__ uint32_t bins[kBinCopies][kBins];
  __shared__ uint32_t scan_lds[2][kSelectWaves], found[2], holes_lds[kSelectWaves];
  const int t = threadIdx.x, wave = t >> 6, row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  SelectRow r;
  const bool longer = select_row<kSelectThreads>(a, row, part, a.parts, &r);
  if (PASS == 0 && part == 0) {
    open_row<kSelectThreads>(a, row, r);
    if (!longer) leave_row<kSelectThreads>(a, row, r);
  }
  if (!longer) return;
  const SplitRow s = split_row(a, row);
  uint32_t least = 0, need = r.places;
  if constexpr (PASS == 2) {
    least = s.state[0];
    need = s.state[1];
  }
  for (int i = t; i < kBinCopies * kBins; i += kSelectThreads) (&bins[0][0])[i] = 0;
  float x[kSelectLoads];
  r.preload(x);
  uint32_t holes;      // (of this part; behind the first launch of the row)
  if constexpr (PASS == 0) {
    const uint32_t mine = find_holes(a, r, r.from, r.to);
    if (r.lane == 0) holes_lds[wave] = mine;
    __syncthreads();
    holes = all_holes<kSelectWaves>(holes_lds);
    if (t == 0) s.state[4 + 2 * a.parts + part] = holes;
    if (r.places == 0) return;
  } else {
    holes = split_holes(a, s);
    if (holes & kHoleInTheWay) {
      if (PASS == 1 && part == 0) leave_row<kSelectThreads>(a, row, r);
      return;
    }
    if (r.places == 0) return;
    split_digit(a, s, PASS - 1, part, least, need, scan_lds, found);
    __syncthreads();
  }
  uint32_t* const mine = bins[wave % kBinCopies];
  if (holes == 0)
    count_digits<PASS, false>(r, x, least, mine);
  else
    count_digits<PASS, true>(r, x, least, mine);
  __syncthreads();
  uint32_t* const to = s.counts + ((int64_t)PASS * a.parts + part) * kBins;
  for (int i = t; i < digit_values(PASS); i += kSelectThreads) {
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < kBinCopies; ++k) n += bins[k][i];
    to[i] = n;
  }
}

template <bool HOLES>
__device__ __forceinline__ void keep_part(const SelectRow& r, float (&x)[kSelectLoads], uint32_t least, uint32_t need,
                                          uint32_t before_sure, uint32_t before_equal, uint32_t (*counts_lds)[kSelectWaves]) {
  uint32_t sure = 0, equal = 0;
  r.walk(x, true, [&](int j, bool real, float v) {
    const uint32_t key = order_key(v);
    const bool middle = r.template earns<HOLES>(j, real) && r.places > 0;
    sure += (uint32_t)__popcll(__ballot(r.given(j, real) || (middle && key > least)));
    equal += (uint32_t)__popcll(__ballot(middle && key == least));
  });
  counts_before(sure, equal, counts_lds);
  write_kept<HOLES>(r, x, least, need, before_sure + sure, before_equal + equal);
}

__global__ __launch_bounds__(kSelectThreads) void kv_select_keep_kernel(const KvEvictArgs a) {
  __shared__ uint32_t scan_lds[2][kSelectWaves], counts_lds[2][kSelectWaves], found[2];
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  SelectRow r;
  if (!select_row<kSelectThreads>(a, row, part, a.parts, &r)) return;
  const SplitRow s = split_row(a, row);
  uint32_t least = 0, need = r.places;
  uint32_t before_sure = 0, before_equal = 0;      // kept in the parts before this one
  float x[kSelectLoads];
  r.preload(x);
  const uint32_t holes = split_holes(a, s);
  if (holes & kHoleInTheWay) return;
  if (r.places > 0) {
    least = s.state[2];
    need = s.state[3];
    before_sure = s.state[4 + part] + s.state[4 + a.parts + part];
    const PartsBefore before = split_digit(a, s, 2, part, least, need, scan_lds, found);
    before_sure += before.above;
    before_equal = before.equal;
  }
  // (the ends before this part's stretch are kept as well)
  const int stretch = (r.len + 64 * a.parts * kSelectWaves - 1) / (64 * a.parts * kSelectWaves) * 64;
  const int begin = min(r.len, part * kSelectWaves * stretch);
  before_sure += (uint32_t)(min(begin, r.lo) + max(0, begin - r.hi));
  if (holes == 0)
    keep_part<false>(r, x, least, need, before_sure, before_equal, counts_lds);
  else
    keep_part<true>(r, x, least, need, before_sure, before_equal, counts_lds);
}

// The compaction.  A batch is 64 KB of rows that become neighbours: the keys or the values
// of a head, kept[j] -> j for `rows` successive j.  A workgroup reads its batch into
// registers, says so, and writes once every batch that reads what it overwrites has been
// read.  kept[j] >= j grows with j, so those are earlier batches of the same list; the
// workgroups of a list take its batches in the order in which they start, and say that
// they have read without waiting for anything: every wait ends.
// Bound by the rows read and written (64 sequences of 8 heads of 128 to 2048 positions: 1.07 GB
// in 214 us, 5.0 TB/s; a copy of that size reaches 5.2), past the caches: nothing is used twice.
// Batches of 32 KB are 2 to 8 % behind, rows that stay in the caches 5 %.
constexpr int kMoveLoads = 8;       // of 16 bytes a thread
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_move_kernel(const KvEvictArgs a) {
  __shared__ uint32_t ticket_lds;
  const int t = threadIdx.x;
  const int list = blockIdx.x % (2 * a.B * a.Hkv);
  const int which = list & 1, bh = list >> 1, b = bh / a.Hkv, h = bh % a.Hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const int new_len = a.new_lens[b];
  if (len <= a.budget || new_len != a.budget) return;     // (not cut)
  uint32_t* const taken = a.order + (int64_t)list * (1 + a.batches);
  uint32_t* const read = taken + 1;
  if (t == 0) ticket_lds = __hip_atomic_fetch_add(taken, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const int batch = (int)ticket_lds;
  char* const cache = (char*)(which ? a.v_cache : a.k_cache) + (int64_t)h * a.head_stride;
  const int32_t* const kept = a.kept + (int64_t)bh * a.budget;
  const int32_t* const pages = a.table + (int64_t)b * a.table_stride;
  const int pieces = a.row_bytes / 16, rows = (kMoveLoads * THREADS) / pieces;
  const int first = batch * rows, last = min(a.budget, first + rows);     // rows that are written
  // Three rounds of loads, each of them all at once: the old places, the pages, the rows.  (A lane
  // without a row, or with one that stays, reads a valid one and writes nothing.)
  int dst[kMoveLoads], src[kMoveLoads], piece[kMoveLoads];
  int dst_page[kMoveLoads], src_page[kMoveLoads];
  bool moves[kMoveLoads];
#pragma unroll
  for (int i = 0; i < kMoveLoads; ++i) {
    const int e = i * THREADS + t, in_batch = divided(e, a.by_pieces);
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
    const int64_t at = there ? (int64_t)src_page[i] * a.page_stride + (int64_t)slot * a.slot_stride : 0;
    x[i] = __builtin_nontemporal_load((const u32x4*)(cache + at + piece[i] * 16));
  }
  // The rows' sums go with the keys.
  const bool with_sums = which == 0;
  const float* const sums = a.sums + (int64_t)b * a.sums_stride_b + (int64_t)h * a.sums_stride_h;
  float* const sums_out = a.sums_out + (int64_t)b * a.out_stride_b + (int64_t)h * a.out_stride_h;
  float sum[kMoveLoads];
  if (with_sums) {
#pragma unroll
    for (int i = 0; i < kMoveLoads; ++i)
      if (i * THREADS < rows) sum[i] = sums[kept[min(first + i * THREADS + t, last - 1)]];
  }
  // Every read of the batch has arrived: the rows are in registers, and nobody reads in this
  // kernel what another workgroup writes, so that the words need no cache to be written
  // back or invalidated (relaxed, but seen by the whole card).
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (t == 0) __hip_atomic_store(read + batch, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // earlier batches with a source among the rows first .. last - 1 (and, before the sums behind the
  // last row are cleared, those with a source there)
  const bool clears = with_sums && batch == a.batches - 1;
  for (int c = t; c < batch; c += THREADS) {
    const int c_last = kept[c * rows + rows - 1];
    if ((kept[c * rows] < last && c_last >= first) || (clears && c_last >= a.budget))
      while (__hip_atomic_load(read + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) __builtin_amdgcn_s_sleep(2);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMoveLoads; ++i) {
    const int slot = dst[i] - divided(dst[i], a.by_page) * a.page_size;
    const int64_t at = (int64_t)dst_page[i] * a.page_stride + (int64_t)slot * a.slot_stride;
    if (moves[i]) __builtin_nontemporal_store(x[i], (u32x4*)(cache + at + piece[i] * 16));
  }
  if (with_sums) {
#pragma unroll
    for (int i = 0; i < kMoveLoads; ++i) {
      const int j = first + i * THREADS + t;
      if (i * THREADS < rows && i * THREADS + t < rows && j < last) sums_out[j] = sum[i];
    }
    if (clears)
      for (int j = a.budget + t; j < len; j += THREADS) sums_out[j] = 0.0f;
  }
}

}  // namespace

void launch_kv_append(const KvAppendArgs& args, int kind, hipStream_t stream) {
  KvAppendArgs a = args;
  const bool fp8 = kind == kKvFp8Bf16 || kind == kKvFp8F16;
  a.pieces = a.D / 8;
  a.by_page = fast_div(a.page_size);
  a.by_pieces = fast_div(a.pieces);
  a.by_token = fast_div(a.Hkv * a.pieces);
  const int64_t items = (int64_t)a.tokens * a.Hkv * a.pieces;
  const dim3 grid((unsigned)((items + 255) / 256)), block(256);
  const int bf16 = kind == kKvBf16 || kind == kKvFp8Bf16;
  if (fp8)
    hipLaunchKernelGGL((kv_append_kernel<true>), grid, block, 0, stream, a, bf16);
  else
    hipLaunchKernelGGL((kv_append_kernel<false>), grid, block, 0, stream, a, bf16);
}

int kv_evict_move_threads(int budget, int row_bytes) {
  // A head's rows that fit a batch of 16 KB need no larger workgroup: 13952 lists of 43 rows of 128
  // bytes in 43 us (512 threads, with room for twelve times the rows: 124), 6848 of 41 in 27 (65).
  return (int64_t)budget * row_bytes <= kMoveLoads * kKvMoveFewThreads * 16 ? kKvMoveFewThreads : kKvMoveThreads;
}

int kv_evict_batches(int budget, int row_bytes) {
  const int rows = kMoveLoads * kv_evict_move_threads(budget, row_bytes) / (row_bytes / 16);
  return (budget + rows - 1) / rows;
}

int kv_evict_parts(int rows, int max_len) {
  // One workgroup takes 9 us for a row of 2304 positions, 20 for 16384, 33 for 32768 and 58 for 65536,
  // whatever their number up to 192; the four launches 30, 31 and 39 us at 32768 and 33, 40 and 59 at
  // 65536 for 32, 64 and 128 rows (and 25 and more below).
  if (max_len <= 32768 || rows > 64) return 1;
  const int most = (max_len + 4095) / 4096;
  return min(min(256 / rows, most), kMostParts);
}

// A row of 2048 sums is in the registers of 256 threads, which cost less to start and to bring to a
// barrier, and more rows share a CU: 6976 rows of up to 64 sums in 27 us (1024 threads: 99), 3424 of
// up to 927 in 23 (64), 1024 of up to 600 in 10 (20), 128 in 7.9 (8.2), 8 of 2000 in 10.1 (9.4).
// Past that a few threads have to read a row again for each digit, which pays as long as other rows
// hide it: 576 rows of up to 4000 in 17 (20), but of 8000 in 26 (23); 1024 of 5000 in 22 (28) and of
// 9000 in 32 (40), but of 16000 in 60 (56); 256 of 2300 in 12.1 (10.8).
static int select_threads(int rows, int max_len) {
  return max_len <= kSelectLoads * kFewThreads || max_len <= std::min<int64_t>(8 * (int64_t)rows, kSelectLoads * kSelectThreads)
             ? kFewThreads : kSelectThreads;
}

size_t kv_evict_workspace_bytes(int rows, int row_bytes, int max_len, int budget) {
  const size_t order = 2 * (size_t)rows * (1 + kv_evict_batches(budget, row_bytes));
  const int parts = kv_evict_parts(rows, max_len);
  return 4 * (order + (parts > 1 ? (size_t)rows * kv_split_words(parts) : 0));
}

void launch_kv_evict(const KvEvictArgs& args, hipStream_t stream) {
  KvEvictArgs a = args;
  const int rows = a.B * a.Hkv;
  a.by_page = fast_div(a.page_size);
  a.by_pieces = fast_div(a.row_bytes / 16);
  a.batches = kv_evict_batches(a.budget, a.row_bytes);
  a.parts = kv_evict_parts(rows, a.max_len);
  a.split = a.order + 2 * (size_t)rows * (1 + a.batches);
  if (a.parts == 1 && select_threads(rows, a.max_len) == kFewThreads) {
    hipLaunchKernelGGL((kv_select_kernel<kFewThreads>), dim3(rows), dim3(kFewThreads), 0, stream, a);
  } else if (a.parts == 1) {
    hipLaunchKernelGGL((kv_select_kernel<kSelectThreads>), dim3(rows), dim3(kSelectThreads), 0, stream, a);
  } else {
    const dim3 grid(rows * a.parts), block(kSelectThreads);
    hipLaunchKernelGGL((kv_select_digit_kernel<0>), grid, block, 0, stream, a);
    hipLaunchKernelGGL((kv_select_digit_kernel<1>), grid, block, 0, stream, a);
    hipLaunchKernelGGL((kv_select_digit_kernel<2>), grid, block, 0, stream, a);
    hipLaunchKernelGGL(kv_select_keep_kernel, grid, block, 0, stream, a);
  }
  const dim3 batches(2 * rows * a.batches);
  if (kv_evict_move_threads(a.budget, a.row_bytes) == kKvMoveThreads)
    hipLaunchKernelGGL((kv_move_kernel<kKvMoveThreads>), batches, dim3(kKvMoveThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((kv_move_kernel<kKvMoveFewThreads>), batches, dim3(kKvMoveFewThreads), 0, stream, a);
}

}  // namespace vk

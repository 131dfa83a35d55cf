// paged_attention.hip — the attention of one new token over a paged key-value cache.
//
// For a query head h on key/value head g and the positions j that it sees,
//   s_j = scale k_scale_g q_h . k_j   (c tanh(s_j / c) with a softcap c),
//   out_h = v_scale_g (sum_j e^{s_j} v_j) / (sum_j e^{s_j} + e^{sink_h}),
// in one pass over keys and values: a running reference m (at least the maximum less 8 in
// powers of two), the sum of 2^{s log2 e - m} and the weighted sum of the values, both
// rescaled when m rises; partial results with references m_p join as sum_p 2^{m_p - m} (.).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attention_math.hpp"
#include "fast_div.hpp"
#include "paged_attention.hpp"
#include "paged_attention_layout.hpp"

namespace vk {
namespace {

using namespace attention;

constexpr int kAhead = 4;    // value tiles that are read from LDS ahead of their products

// Maximum / sum over the four lanes l % 16, + 16, + 32, + 48 that hold a head's column.
__device__ __forceinline__ float over_column_max(float x) {
  const uint32_t u = __float_as_uint(x);
  u32x2 s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float over_column_sum(float x) {
  const uint32_t u = __float_as_uint(x);
  u32x2 s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// What a work item (16 heads of one sequence) sees of its cache: positions [lo, len) and, in front of a window,
// [0, first).  It walks along a line of `walk` places, the first `split` of them the positions at the beginning,
// the others positions `shift` further on (where the two parts meet or nearly do, all positions are
// walked, those between hidden).
struct Span {
  int lo, len, first;
  int split, shift, walk;
  int units;   // of kPaUnit places; at least one
  __device__ __forceinline__ int position(int place) const { return place < split ? place : place + shift; }
};
__device__ __forceinline__ Span span_of(int len, const PagedAttentionArgs& a) {
  Span s;
  s.len = min(max(len, 0), a.max_len);
  s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
  s.first = min(a.keep_first, s.lo);
  s.split = (s.first + kPaUnit - 1) & ~(kPaUnit - 1);   // a whole number of units
  s.shift = (s.lo & ~15) - s.split;
  if (s.shift <= 0 && s.first > 0) s.split = s.shift = 0;
  s.walk = s.len - s.shift;
  s.units = max(1, (s.walk + kPaUnit - 1) / kPaUnit);
  return s;
}

// Workgroups of a CU (wavefronts of a SIMD), by the registers that a width needs: the grid is as
// many as the card holds at once.
constexpr int residents(int DP) { return DP <= 128 ? 2 : 1; }

struct KernelArgs {
  PagedAttentionArgs a;
  PagedAttentionPlan p;
  FastDiv by_page;       // position / page_size
  FastDiv by_block;      // slot of a page / positions with one scale
};

__device__ __forceinline__ int page_of(const KernelArgs& A, int pos) { return divided(pos, A.by_page); }

// Places of a span, at most.  (Any window may be asked for: nothing is added in 32 bits to one that reaches
// beyond max_len.)
int most_seen(int max_len, int window, int keep_first) {
  if (window <= 0) return max_len;
  const int64_t split = ((int64_t)std::min(keep_first, max_len) + kPaUnit - 1) / kPaUnit * kPaUnit;
  return (int)std::min<int64_t>(max_len, (int64_t)window + 16 + split);
}

// The units of all items in order (sequence, head item, unit), cut into equal shares.
struct Share {
  int first, last;   // units of this workgroup, of those of its group
  int per;           // units of a share
  int b, unit0;      // the sequence that `first` lies in, and its first unit
  int group, index;  // head tile (where those have workgroups of their own; else 0), workgroup of it
};

// Inclusive sum over the lanes of a wavefront up to this one.
__device__ __forceinline__ int lanes_up_to(int x) {
#define VK_ADD_FROM(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, true)
  VK_ADD_FROM(0x111, 0xF);   // the lane 1, 2, 4, 8 below, within rows of 16
  VK_ADD_FROM(0x112, 0xF);
  VK_ADD_FROM(0x114, 0xF);
  VK_ADD_FROM(0x118, 0xF);
  VK_ADD_FROM(0x142, 0xA);   // lane 15 of rows 0 and 2 to rows 1 and 3
  VK_ADD_FROM(0x143, 0xC);   // lane 31 to rows 2 and 3
#undef VK_ADD_FROM
  return x;
}

// Every wavefront finds its workgroup's share by itself from the lengths: a lane adds up the units of
// B / 64 sequences, a scan over the lanes finds the lane that holds `first`, which walks on.  (No
// LDS and no barrier: this is all latency, in front of the first load of a key.)
__device__ __forceinline__ bool find_share(const KernelArgs& A, Share* sh) {
  const PagedAttentionArgs& a = A.a;
  const int lane = threadIdx.x & 63;
  const int heads = a.Hkv * (A.p.head_tiles / A.p.tile_groups);
  sh->group = (int)blockIdx.x / A.p.group_workgroups;
  sh->index = (int)blockIdx.x - sh->group * A.p.group_workgroups;
  if (sh->group >= A.p.tile_groups) return false;   // (uniform over the workgroup, as below)
  const int per = (a.B + 63) / 64;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < a.B) mine += span_of(a.lens[b], a).units;
  }
  const int scan = lanes_up_to(mine);
  const int total = __builtin_amdgcn_readlane(scan, 63) * heads;
  const int share = max(A.p.min_units, (total + A.p.group_workgroups - 1) / A.p.group_workgroups);
  const int first = sh->index * share;
  if (first >= total) return false;
  int at = (scan - mine) * heads, b = lane * per;
  const bool here = first >= at && first < at + mine * heads;
  if (here && per > 1) {
    for (;; ++b) {
      const int units = span_of(a.lens[b], a).units * heads;
      if (first < at + units) break;
      at += units;
    }
  }
  const int owner = (int)__builtin_ctzll(__ballot(here));
  sh->first = first;
  sh->last = min(total, first + share);
  sh->per = share;
  sh->b = __builtin_amdgcn_readlane(b, owner);
  sh->unit0 = __builtin_amdgcn_readlane(at, owner);
  return true;
}

template <class M, bool FP8, int DP>
struct Tile {
  static constexpr int kElem = FP8 ? 1 : 2;
  static constexpr int kRowBytes = DP * kElem;
  static constexpr int kPieces = pa_value_pieces(kRowBytes);   // lanes that load a value row
  static constexpr int kRowsPerLoad = 64 / kPieces;
  static constexpr int kVLoads = kPaWaveRows / kRowsPerLoad;
  static constexpr int kPitch = kPieces * 16;            // bytes of a row in LDS
  static constexpr int kKLoads = pa_key_loads(kRowBytes);   // 64 bytes of 16 rows each
  static constexpr int kSteps = DP / 32;                 // MFMAs over the head's width
  static constexpr int kOutPitch = DP + 4;               // floats of a head's sums in LDS
  static constexpr int kWaveLds = kPaWaveRows * kPitch > kPaHeads * kOutPitch * 4
                                      ? kPaWaveRows * kPitch : kPaHeads * kOutPitch * 4;
};

// The attention itself.  A work item is 16 query heads on one key/value head of one sequence; a
// workgroup has an even share of all items' units (128 positions) and walks through the items in
// it, or one whole item where the call is short.  A wavefront takes 32 positions at a time, by itself:
//   S = K q^T      (16 x 16 x 32, keys the first operand: a lane holds one head's scores of 8
//                   positions, and running maximum, sum and rescaling stay in the lane),
//   O^T += V^T P^T (the weights are in the lane that the second product wants them in; the
//                   values go to LDS by rows and come back transposed, 4 x 16 at a time).
// The four wavefronts' results meet in LDS at an item's end, several workgroups' in the joining
// kernel.  The matrix cores run at 1 % of their rate and a CU issues some 170 vector instructions
// a tile: the stream of keys and values bounds it.  One sequence of 131071 positions, 8 heads of
// 128: 88 us for 537 MB, 6.1 TB/s (a kernel that only reads reaches 7.0); 255 sequences on an
// 8-bit cache, 2.34 GB: 373 us, 6.3 TB/s; 64 sequences of 64-wide heads, the cache token by
// token, 563 MB: 106 us, 5.3 TB/s (head by head 96 us).  5.6 us of each are start, length,
// page, first tile and the way out.  Registers: with fewer than 256 a lane (three workgroups a
// CU) a 128-wide head spills (131 us where two take 97), a 64-wide one gains nothing.
// FULL: D is DP.  P16: pages are multiples of 16 positions, so that a page is the same for 16 rows.
// SCALES: an 8-bit cache's blocks of positions have scales of their own.  A lane loads the scale of one
// position's keys or values with the tile; scores are multiplied by the keys', the weights by the values'
// before they become 16-bit terms (in bf16 whatever the queries' type: codes are exact in it, and a weight
// times a scale needs its range).  255 sequences of up to 8192 positions, 8 heads of 4 of 128, scales for 16 positions
// each: 376 us for 2.35 GB, as with a scale for each head; one of 131071: 42 us for 269 MB, 6.3 TB/s.
template <class M, bool FP8, int DP, bool P16, bool FULL, bool SCALES>
__global__ __launch_bounds__(256, residents(DP)) void paged_attention_kernel(const KernelArgs A) {
  typedef Tile<M, FP8, DP> L;
  typedef typename M::V8 V8;
  typedef std::conditional_t<SCALES, Bf16, M> W;      // what weights and values are multiplied in
  const PagedAttentionArgs& a = A.a;
  __shared__ __attribute__((aligned(16))) char lds[kPaWaves * L::kWaveLds];
  __shared__ __attribute__((aligned(16))) float scale_lds[SCALES ? kPaWaves : 1][2 * kPaWaveRows];
  __shared__ float wave_m[kPaWaves][kPaHeads], wave_l[kPaWaves][kPaHeads];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int tiles = A.p.head_tiles / A.p.tile_groups, item_heads = a.Hkv * tiles;   // of a sequence, in the group
  char* const my_lds = lds + wave * L::kWaveLds;

  Share sh;
  int item_in_b = 0;
  u32x4* const ends_here = (u32x4*)((char*)a.workspace + A.p.ends_at) + blockIdx.x;
  if (A.p.workgroups > 0) {
    if (!find_share(A, &sh)) {
      if (threadIdx.x == 0) *ends_here = u32x4{0, 0, 0, 0};
      return;
    }
  } else {
    sh.first = sh.group = 0;
    sh.b = blockIdx.x / item_heads;
    item_in_b = blockIdx.x % item_heads;
  }
  const ConstInts lens = read_only(a.lens);
  Span span = span_of(lens[sh.b], a);
  int unit_at;         // unit of the item that the segment begins with
  int left;            // units of the share that are left
  if (A.p.workgroups > 0) {
    const int in_b = sh.first - sh.unit0;
    item_in_b = in_b / span.units;
    unit_at = in_b % span.units;
    left = sh.last - sh.first;
  } else {
    unit_at = 0;
    left = span.units;
  }
  int b = sh.b;
  int item_unit0 = A.p.workgroups > 0 ? sh.first - unit_at : 0;   // the item's first unit
  auto item_at = [&](int b, int in_b) { return (b * a.Hkv + in_b / tiles) * A.p.head_tiles + sh.group + in_b % tiles; };
  if (A.p.workgroups > 0 && threadIdx.x == 0) {
    // For the join: the item that other workgroups began and this one ends, if there is one.
    const bool ends = unit_at > 0 && span.units - unit_at <= left;
    const int begun = item_unit0 / sh.per;
    *ends_here = u32x4{(uint32_t)item_at(b, item_in_b), (uint32_t)((int)blockIdx.x - sh.index + begun),
                       ends ? (uint32_t)(sh.index - begun + 1) : 0u, 0u};
  }

  const int64_t slot_bytes = a.slot_stride * L::kElem, page_bytes = a.page_stride * L::kElem;
  while (left > 0) {
    const int units = min(left, span.units - unit_at);
    const int g = item_in_b / tiles, head0 = (sh.group + item_in_b % tiles) * kPaHeads;
    const int heads = min(kPaHeads, a.G - head0);
    const ConstInts pages = read_only(a.table + (int64_t)b * a.table_stride);
    const char* const kbase = (const char*)a.k_cache + (int64_t)g * a.head_stride * L::kElem;
    const char* const vbase = (const char*)a.v_cache + (int64_t)g * a.head_stride * L::kElem;

    // The queries as the MFMA's second operand: lane (col, quad) holds head col and, of
    // every 32 values, the 8 at 8 quad (of an 8-bit cache: of every 64 the 16 at 16 quad,
    // in two operands; the keys below are dealt out alike).
    V8 q[L::kSteps];
    {
      // (a lane without a head or past the width reads the first values instead)
      const int64_t head = (int64_t)(g * a.G + head0 + min(col, heads - 1)) * a.q_stride_h;
      const char* const row = (const char*)a.q + ((int64_t)b * a.q_stride_b + head) * 2;
#pragma unroll
      for (int i = 0; i < L::kSteps; ++i) {
        const int d = FP8 ? (i / 2) * 64 + quad * 16 + (i % 2) * 8 : i * 32 + quad * 8;
        const u32x4 x = *(const u32x4*)(row + (d < a.D ? d : 0) * 2);
        q[i] = as_v8<M>(col < heads && d < a.D ? x : u32x4{0, 0, 0, 0});
      }
    }
    const float k_scale = !SCALES && a.k_scale != nullptr ? a.k_scale[g] : 1.0f;
    const float to_log2 = a.scale * k_scale * kLog2e;
    const float cap_in = a.softcap > 0.0f ? 2.0f * a.scale * k_scale * kLog2e / a.softcap : 0.0f;
    const float cap_out = a.softcap * kLog2e;

    f32x4 acc[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) acc[i] = f32x4{0, 0, 0, 0};
    float m = kNegInf, l = 0.0f;

    u32x4 kreg[2][L::kKLoads], vreg[L::kVLoads];
    const int begin = unit_at * kPaUnit + wave * kPaWaveRows;        // places
    const int end = min((unit_at + units) * kPaUnit, span.walk);   // no tile is wholly behind it

    // The table's entries of a tile, asked for a tile ahead of the loads that need them (one for
    // each 16 positions where pages are multiples of 16 long, else one a lane: position lane % 32);
    // -1 behind the length.  The last entry stands in for those that the table does not have.
    const int last_entry = page_of(A, max(span.len - 1, 0));
    int ids[2] = {-1, -1};
    auto ask_pages = [&](int pos0) {
      if constexpr (P16) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int id = pages[min(page_of(A, pos0 + 16 * t), last_entry)];
          ids[t] = pos0 + 16 * t < span.len ? id : -1;
        }
      } else {
        const int pos = pos0 + (lane & 31);
        const int id = (a.table + (int64_t)b * a.table_stride)[min(page_of(A, pos), last_entry)];
        ids[0] = (pos >= span.lo || pos < span.first) && pos < span.len ? id : -1;
      }
    };
    // Of the tile that is loaded: its pages (P16), or where the lane's position lies.
    int page0 = -1, page1 = -1;
    int64_t half_at[2] = {0, 0};     // bytes from the cache's start to positions 0 and 16 of the tile
    int64_t row_at = 0;
    bool row_ok = false;
    // The scale of position lane % 32 of the tile that is loaded: of its keys, or in the upper lanes of its values
    // (1 where the position does not count: what is stored there may be anything).
    float scale_of_row = 1.0f;
    const float* const scales = lane < 32 ? a.k_scale : a.v_scale;
    auto load_scale = [&](int page, int slot, bool there) {
      const int64_t at = ((int64_t)page * a.Hkv + g) * a.scale_blocks + divided(slot, A.by_block);
      scale_of_row = there ? scales[at] : 1.0f;
    };
    auto take_pages = [&](int pos0) {
      if constexpr (P16) {
        page0 = (uint32_t)ids[0] < (uint32_t)a.num_pages ? ids[0] : -1;
        page1 = (uint32_t)ids[1] < (uint32_t)a.num_pages ? ids[1] : -1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int pos = pos0 + 16 * t;
          half_at[t] = (int64_t)max(t == 0 ? page0 : page1, 0) * page_bytes +
                       (uint32_t)(pos - page_of(A, pos) * a.page_size) * (uint64_t)(uint32_t)slot_bytes;
        }
        if constexpr (SCALES) {
          const int half = lane & 16, pos = pos0 + half, page = half ? page1 : page0;
          load_scale(page, pos - page_of(A, pos) * a.page_size + col,
                     page >= 0 && pos + col < span.len && (pos + col >= span.lo || pos + col < span.first));
        }
      } else {
        const int pos = pos0 + (lane & 31);
        row_ok = (uint32_t)ids[0] < (uint32_t)a.num_pages;
        row_at = row_ok ? (int64_t)ids[0] * page_bytes + (int64_t)(pos - page_of(A, pos) * a.page_size) * slot_bytes : 0;
        if constexpr (SCALES) load_scale(ids[0], pos - page_of(A, pos) * a.page_size, row_ok);
      }
    };
    // Where a row of the loaded tile lies (generic pages), from the lane that looked it up.
    auto row_from = [&](int row) -> int64_t {
      const int lo = __shfl((int)(uint32_t)row_at, row);
      const int hi = __shfl((int)(row_at >> 32), row);
      return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
    };
    // What lies behind a row's last value is taken as zeros (keys) or not used (values), and such lanes
    // read the row's first bytes instead.
    const int row_bytes = FULL ? L::kRowBytes : a.D * L::kElem;
    auto key_piece = [&](const char* row, int i) -> u32x4 {
      const int at = pa_key_at(quad, i);
      const u32x4 x = *(const u32x4*)(row + pa_piece_at(at, row_bytes));
      return at < row_bytes ? x : u32x4{0, 0, 0, 0};
    };
    const int piece = lane % L::kPieces, sub = lane / L::kPieces;
    const uint32_t value_at = pa_value_at(piece, row_bytes);
    const uint32_t key_lane = (uint32_t)col * (uint32_t)slot_bytes, value_lane = (uint32_t)sub * (uint32_t)slot_bytes + value_at;
    auto load_k = [&] {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char* const row = P16 ? kbase + half_at[t] + key_lane : kbase + row_from(16 * t + col);
#pragma unroll
        for (int i = 0; i < L::kKLoads; ++i) kreg[t][i] = key_piece(row, i);
      }
    };
    // (Values past the caches: with up to 16 heads nobody reads them again, and the keys' lines, which two loads share, then
    // stay until the second: 97 -> 87 us for 131071 positions of 8 heads of 128.  Keys past the
    // caches too cost a fifth at rows of 128 bytes.  Of more heads' tiles the later ones would gain 5 to
    // 10 % by values that stay, and lose as much where scores are kept.)
    auto load_v = [&] {
#pragma unroll
      for (int i = 0; i < L::kVLoads; ++i) {
        constexpr int kHalf = L::kVLoads / 2;
        const char* from;
        if constexpr (P16)
          from = vbase + (half_at[i / kHalf] + (int64_t)(i % kHalf * L::kRowsPerLoad) * slot_bytes) + value_lane;
        else
          from = vbase + row_from(i * L::kRowsPerLoad + sub) + value_at;
        vreg[i] = __builtin_nontemporal_load((const u32x4*)from);
      }
    };

    // One tile; with MORE behind it, the next one's keys are asked for as soon as this one's have
    // been multiplied, its values as soon as this one's are in LDS.
    auto tile = [&](int place, auto more) {
      constexpr bool MORE = decltype(more)::value;
      const int pos0 = span.position(place);
      if constexpr (SCALES) scale_lds[wave][lane] = scale_of_row;
      // which of the 8 positions of this lane count, and which value rows it loaded do
      bool whole;
      uint32_t rows;        // bit r: position pos0 + r counts
      if constexpr (P16) {
        whole = (pos0 >= span.lo || pos0 + 32 <= span.first) && pos0 + 32 <= span.len && page0 >= 0 && page1 >= 0;
        rows = 0xFFFFFFFFu;
        if (!whole) {
          if (page0 < 0) rows &= 0xFFFF0000u;
          if (page1 < 0) rows &= 0x0000FFFFu;
          const int n = span.len - pos0, skip = span.lo - pos0, kept = span.first - pos0;
          if (n < 32) rows &= n <= 0 ? 0u : (1u << n) - 1u;
          if (skip > 0) rows &= (skip >= 32 ? 0u : ~0u << skip) | (kept <= 0 ? 0u : kept >= 32 ? ~0u : (1u << kept) - 1u);
        }
      } else {
        rows = (uint32_t)__ballot(row_ok);
        whole = rows == 0xFFFFFFFFu;
      }

      f32x4 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x4{0, 0, 0, 0};
        if constexpr (FP8) {
#pragma unroll
          for (int i = 0; i < L::kKLoads; ++i) {
            s[t] = M::mfma(fp8x8<M>(kreg[t][i][0], kreg[t][i][1]), q[2 * i], s[t]);
            s[t] = M::mfma(fp8x8<M>(kreg[t][i][2], kreg[t][i][3]), q[2 * i + 1], s[t]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < L::kKLoads; ++i) s[t] = M::mfma(as_v8<M>(kreg[t][i]), q[i], s[t]);
        }
      }
      if constexpr (MORE) {
        take_pages(span.position(place + kPaUnit));
        load_k();
        ask_pages(span.position(place + 2 * kPaUnit));
      }

      // scores in powers of two
      float x[8];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[t * 4 + r] = s[t][r];
      f32x4 value_scale[2];
      if constexpr (SCALES) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const f32x4 key_scale = *(const f32x4*)&scale_lds[wave][t * 16 + quad * 4];
          value_scale[t] = *(const f32x4*)&scale_lds[wave][kPaWaveRows + t * 16 + quad * 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) x[t * 4 + r] *= key_scale[r];
        }
      }
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = capped(x[i] * cap_in, cap_out);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= to_log2;
      }
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!((rows >> (t * 16 + quad * 4 + r)) & 1u)) x[t * 4 + r] = kNegInf;
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      top = over_column_max(top);
      if (__any(top > m + kSlack)) {
        const float m_new = fmaxf(m, top);
        const float fix = exp2_fast(m - or_zero(m_new));
        m = m_new;
        l *= fix;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) acc[i] *= fix;
      }
      // The weights as two 16-bit terms: 16 bits of each weight instead of 8 (the matrix
      // cores idle otherwise), so that the result is off by its own rounding alone.  Terms in fp16 end at
      // 2^-24, so that many positions far below one of large weight would be lost: there a tile's weights
      // are taken relative to its own maximum, as 2^15 of it, and what they sum to is brought to the
      // reference in 32 bits (131071 positions of 8 heads of 128: 94.3 us with and 94.2 without).
      const float ref = W::kTileScale ? or_zero(top) - 15.0f : or_zero(m);
      const float to_ref = top == kNegInf ? 0.0f : exp2_fast(ref - m);
      float sum = 0.0f;
      union { typename W::T e[8]; typename W::V8 v; } hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float p = exp2_fast(x[i] - ref);
        if constexpr (W::kTileScale) sum += p; else l += p;
        if constexpr (SCALES) p *= value_scale[i / 4][i % 4];
        hi.e[i] = (typename W::T)p;
        lo.e[i] = (typename W::T)(p - (float)hi.e[i]);
      }
      if constexpr (W::kTileScale) l += sum * to_ref;
      auto add_values = [&](f32x4& sums, typename W::V8 v) {
        if constexpr (W::kTileScale) {
          sums += to_ref * W::mfma(v, lo.v, W::mfma(v, hi.v, f32x4{0, 0, 0, 0}));
        } else {
          sums = W::mfma(v, hi.v, sums);
          sums = W::mfma(v, lo.v, sums);
        }
      };

      // The values to LDS, row after row (rows that do not count as zeros: what is stored
      // there may be anything), 32-byte pairs of pieces exchanged by the row so that the
      // transposed reads below spread over the banks.
      {
        if (!whole) {
#pragma unroll
          for (int i = 0; i < L::kVLoads; ++i)
            if (!((rows >> (i * L::kRowsPerLoad + sub)) & 1u)) vreg[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < L::kVLoads; ++i) {
          const int row = i * L::kRowsPerLoad + sub;
          const int turn = FP8 ? (L::kPieces >= 16 ? row & 7 : L::kPieces == 8 ? (row >> 1) & 7 & (L::kPieces - 1) : 0)
                               : 2 * (L::kPieces >= 16 ? row & 7 : L::kPieces == 8 ? (row >> 1) & 3 : 0);
          *(u32x4*)(my_lds + row * L::kPitch + ((piece ^ turn) * 16)) = vreg[i];
        }
      }
      // The scores, where the positions' weights are wanted: [16 positions][head][position], so that a
      // wavefront's are one piece.  (75 MB of them beside 2.4 GB of keys and values cost 85 us of 500:
      // the same stores dropped by a range check cost nothing, a quarter of them 36 us, one in eight
      // tiles' 14 us, and neither their cache hints nor their place in the loop change it: it is the
      // memory's price of writes among reads.)
      if (A.p.score_pitch > 0 && col < heads) {
        float* const to = (float*)((char*)a.workspace + A.p.scores_at) + quad * 4 +
                          (((int64_t)(b * a.Hkv + g) * A.p.score_pitch + pos0) * a.G + (head0 + col) * 16);
        if (pos0 + quad * 4 < span.len) *(f32x4*)to = f32x4{x[0], x[1], x[2], x[3]};
        if (pos0 + 16 + quad * 4 < span.len) *(f32x4*)(to + 16 * a.G) = f32x4{x[4], x[5], x[6], x[7]};
      }
      if constexpr (MORE) load_v();
      // (lanes read what other lanes of their wavefront wrote: LDS keeps the order, and so must the compiler)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();

      // Weighted values, transposed: rows of the result are the head's width, columns the
      // heads.  Lane (col, quad) reads value col of every 16 of the positions 4 quad + (0..3)
      // and 16 + 4 quad + (0..3): the order in which the scores' tile left the weights.
      if constexpr (FP8) {
        const int r8 = col >> 1, row = (r8 < 4 ? 0 : 12) + quad * 4 + r8;
        const int turn = L::kPieces >= 16 ? row & 7 : L::kPieces == 8 ? (row >> 1) & 7 & (L::kPieces - 1) : 0;
        const int at = row * L::kPitch + (col & 1) * 8;
#pragma unroll
        for (int i0 = 0; i0 < DP / 16; i0 += kAhead) {
          i32x2 c[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if (i0 + i < DP / 16)
              c[i] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                  (__attribute__((address_space(3))) i32x2*)(my_lds + at + (((i0 + i) ^ turn) * 16)));
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (i0 + i < DP / 16) {
              add_values(acc[i0 + i], fp8x8<W>((uint32_t)c[i][0], (uint32_t)c[i][1]));
            }
          }
        }
      } else {
        const int row = quad * 4 + (col >> 2);
        const int turn = L::kPieces >= 16 ? row & 7 : L::kPieces == 8 ? (row >> 1) & 3 : 0;
        const int at = row * L::kPitch + (col & 3) * 8;
#pragma unroll
        for (int i0 = 0; i0 < DP / 16; i0 += kAhead) {
          union { i16x4 h[2]; typename W::V8 v; } c[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (i0 + i < DP / 16) {
              char* const from = my_lds + at + (((i0 + i) ^ turn) * 32);
              c[i].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)from);
              c[i].h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) i16x4*)(from + 16 * L::kPitch));
            }
          }
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (i0 + i < DP / 16) {
              add_values(acc[i0 + i], c[i].v);
            }
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    if (begin < end) {
      ask_pages(span.position(begin));
      take_pages(span.position(begin));
      load_k();
      ask_pages(span.position(begin + kPaUnit));
      load_v();
      int place = begin;
      for (; place + kPaUnit < end; place += kPaUnit) tile(place, std::true_type{});
      tile(place, std::false_type{});
    }

    // The four wavefronts' sums, joined in LDS.
    l = over_column_sum(l);
    if (quad == 0) {
      wave_m[wave][col] = m;
      wave_l[wave][col] = l;
    }
    if (col < heads) {
      float* to = (float*)my_lds + col * L::kOutPitch + quad * 4;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) *(f32x4*)(to + i * 16) = acc[i];
    }
    __syncthreads();
    const bool begins = unit_at == 0, ends = unit_at + units == span.units;
    const bool alone = begins && ends;
    if (A.p.workgroups > 0 && begins && threadIdx.x == 0) {
      const int count = (item_unit0 + span.units - 1) / sh.per - sh.index + 1;
      ((int64_t*)((char*)a.workspace + A.p.meta_at))[item_at(b, item_in_b)] = ((int64_t)count << 32) | blockIdx.x;
    }
    const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
    const int pairs = a.D / 4;
    for (int e = threadIdx.x; e < heads * pairs; e += 256) {
      const int h = e / pairs, d = (e - h * pairs) * 4;
      float mm = kNegInf;
#pragma unroll
      for (int w = 0; w < kPaWaves; ++w) mm = fmaxf(mm, wave_m[w][h]);
      const int hq = g * a.G + head0 + h;
      // (a sink is one more score whose value is zero)
      const float sink = alone && a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf;
      mm = fmaxf(mm, sink);
      const float ref = or_zero(mm);
      float ll = exp2_fast(sink - ref);
      f32x4 o = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kPaWaves; ++w) {
        const float f = exp2_fast(wave_m[w][h] - ref);
        ll += wave_l[w][h] * f;
        o += f * *(const f32x4*)((float*)(lds + w * L::kWaveLds) + h * L::kOutPitch + d);
      }
      if (alone) {
        const float inv = (ll == 0.0f ? 0.0f : 1.0f / ll) * (!SCALES && a.v_scale != nullptr ? a.v_scale[g] : 1.0f);
        typename M::T* to = (typename M::T*)a.out + ((int64_t)b * a.Hkv * a.G + hq) * a.D + d;
        union { typename M::T e[4]; u32x2 u; } r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r.e[j] = (typename M::T)(o[j] * inv);
        *(u32x2*)to = r.u;
        if (d == 0) {
          if (a.lse != nullptr) a.lse[(int64_t)b * a.Hkv * a.G + hq] = log_of_sum(ref, ll, a.sinks != nullptr ? a.sinks + hq : nullptr);
          if (A.p.score_pitch > 0)
            ((f32x2*)((char*)a.workspace + A.p.stats_at))[(int64_t)b * a.Hkv * a.G + hq] = f32x2{ref, ll};
        }
      } else {
        float* part = (float*)((char*)a.workspace + A.p.part_at) + ((int64_t)slot * kPaHeads + h) * DP + d;
        *(f32x4*)part = o;
        if (d == 0) ((f32x2*)((char*)a.workspace + A.p.ml_at))[slot * kPaHeads + h] = f32x2{mm, ll};
      }
    }

    left -= units;
    item_unit0 += span.units;
    unit_at = 0;
    if (left > 0 && ++item_in_b == item_heads) {
      item_in_b = 0;
      ++b;
      span = span_of(lens[b], a);
    }
    if (left > 0) __syncthreads();   // (the sums are read before the next item's values come)
  }
}

// The slot of partial result p of an item whose first share is workgroup `first`'s.
__device__ __forceinline__ int slot_of(int first, int p) { return 2 * (first + p) + (p == 0 ? 1 : 0); }

// Reference and sum of a head over the partial results of its item (`ml`: of slot 0), the sink
// included; every lane of the wavefront gets them.  `first`: the workgroup whose share begins the item.
__device__ __forceinline__ f32x2 joined_stats(const f32x2* ml, int first, int count, float sink) {
  const int lane = threadIdx.x & 63;
  f32x2 x = {kNegInf, 0.0f};
  if (lane < count) x = ml[slot_of(first, lane) * kPaHeads];
  float m = fmaxf(sink, x[0]);
  for (int p = lane + 64; p < count; p += 64) m = fmaxf(m, ml[slot_of(first, p) * kPaHeads][0]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float ref = or_zero(m);
  float l = (lane == 0 ? exp2_fast(sink - ref) : 0.0f) + x[1] * exp2_fast(x[0] - ref);
  for (int p = lane + 64; p < count; p += 64) {
    const f32x2 y = ml[slot_of(first, p) * kPaHeads];
    l += y[1] * exp2_fast(y[0] - ref);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
  return f32x2{ref, l};
}

// Joins the items that several workgroups had a share of.  Where there are few items (SPLIT 4) a
// block takes one head of an item, and its four wavefronts share the partial results; else a
// block looks at the item that ends in workgroup blockIdx.x / groups' share (there is at most one
// that others began) and takes four of its heads, a wavefront each: a block for every item would
// find nothing to do more often than not.  A lane holds four values of the head; where the width
// leaves lanes over, they take other partial results.
// All latency: the partial results of a first round are asked for before the references are known.
template <class M, int SPLIT>
__device__ __forceinline__ void join_heads(const KernelArgs& A, int padded, int groups, f32x4 (*joined)[64]) {
  const PagedAttentionArgs& a = A.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, turn = SPLIT > 1 ? wave : 0;
  const int row = blockIdx.x / groups, group = blockIdx.x % groups;
  int item, first, count;
  if constexpr (SPLIT > 1) {
    const int64_t mt = ((const int64_t*)((const char*)a.workspace + A.p.meta_at))[row];
    item = row;
    first = (int)(uint32_t)mt;
    count = (int)(mt >> 32);
    if (count <= 1) return;
  } else {
    const u32x4 ends = ((const u32x4*)((const char*)a.workspace + A.p.ends_at))[row];
    item = (int)ends[0];
    first = (int)ends[1];
    count = (int)ends[2];
    if (count == 0) return;
  }
  const int item_heads = a.Hkv * A.p.head_tiles;
  const int b = item / item_heads, in_b = item % item_heads;
  const int g = in_b / A.p.head_tiles, head0 = (in_b % A.p.head_tiles) * kPaHeads;
  const int h = SPLIT > 1 ? group : group * 4 + wave, hq = g * a.G + head0 + h;
  const bool there = h < min(kPaHeads, a.G - head0);
  const f32x2* const ml = (const f32x2*)((const char*)a.workspace + A.p.ml_at) + h;
  const int lanes = padded <= 64 ? 16 : padded <= 128 ? 32 : 64, at_once = 64 / lanes;   // lanes of a row
  const int d = (lane & (lanes - 1)) * 4;
  const float* const part = (const float*)((const char*)a.workspace + A.p.part_at) + (int64_t)h * padded + d;
  const int64_t pitch = (int64_t)kPaHeads * padded;
  f32x4 o = {0, 0, 0, 0};
  f32x2 st = {0, 0};
  if (there) {
    const int p0 = turn * at_once + lane / lanes;
    const bool mine = d < a.D;
    f32x4 x = {0, 0, 0, 0};
    if (mine && p0 < count) x = *(const f32x4*)(part + slot_of(first, p0) * pitch);
    st = joined_stats(ml, first, count, a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf);
    if (mine && p0 < count) {
      o = exp2_fast(ml[slot_of(first, p0) * kPaHeads][0] - st[0]) * x;
#pragma unroll 8
      for (int p = p0 + SPLIT * at_once; p < count; p += SPLIT * at_once)
        o += exp2_fast(ml[slot_of(first, p) * kPaHeads][0] - st[0]) * *(const f32x4*)(part + slot_of(first, p) * pitch);
    }
    for (int across = lanes; across < 64; across <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], across);
  }
  if constexpr (SPLIT > 1) {
    joined[turn][lane] = o;
    __syncthreads();
    if (turn > 0) return;
#pragma unroll
    for (int i = 1; i < SPLIT; ++i) o += joined[i][lane];
  }
  if (!there) return;
  if (lane < lanes && d < a.D) {
    const float inv = (st[1] == 0.0f ? 0.0f : 1.0f / st[1]) *
                      (a.v_scale != nullptr && a.scale_blocks == 0 ? a.v_scale[g] : 1.0f);
    union { typename M::T e[4]; u32x2 u; } r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.e[j] = (typename M::T)(o[j] * inv);
    *(u32x2*)((typename M::T*)a.out + ((int64_t)b * a.Hkv * a.G + hq) * a.D + d) = r.u;
  }
  if (lane == 0 && a.lse != nullptr)
    a.lse[(int64_t)b * a.Hkv * a.G + hq] = log_of_sum(st[0], st[1], a.sinks != nullptr ? a.sinks + hq : nullptr);
}

// Adds up the weights that the positions received: a workgroup for 1024 PER positions of a key/value
// head, a thread for 4 PER.  The scores of the first heads and the sums are asked for before the
// heads' references and sums are known, a wavefront for each head.  Bound by the scores, read
// once, and the sums (64 sequences of up to 16384 positions, 8 heads of 4: 113 MB in 28 us with the
// join, 4.0 TB/s; sums four bytes at a time took 41).
constexpr int kSumHeads = kPaWaves;
template <int PER>
__device__ __forceinline__ void add_weights(const KernelArgs& A, int block, int chunks, f32x2* stats) {
  const PagedAttentionArgs& a = A.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bg = block / chunks, b = bg / a.Hkv, g = bg % a.Hkv, Hq = a.Hkv * a.G;
  const Span span = span_of(read_only(a.lens)[b], a);
  const int at = (block % chunks) * (1024 * PER);       // places
  if (at >= span.walk) return;
  const float* const scores = (const float*)((const char*)a.workspace + A.p.scores_at) +
                              (int64_t)bg * A.p.score_pitch * a.G;
  float* const to = a.sums + (int64_t)b * a.sums_stride_b + (int64_t)g * a.sums_stride_h;
  const int place0 = at + threadIdx.x * 4;        // and PER - 1 more, 1024 apart
  // (16 bytes at a time where the sums' rows allow it and all four positions are seen)
  const bool wide = (reinterpret_cast<uintptr_t>(to) & 15) == 0;
  auto all_seen = [&](int pos) { return wide && (pos >= span.lo || pos + 3 < span.first) && pos + 3 < span.len; };
  float sum[PER][4];
  f32x4 old[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int pos = span.position(place0 + 1024 * k);
    old[k] = f32x4{0, 0, 0, 0};
    if (all_seen(pos)) old[k] = *(const f32x4*)(to + pos);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[k][j] = 0.0f;
  }
  for (int h0 = 0; h0 < a.G; h0 += kSumHeads) {
    const int n = min(kSumHeads, a.G - h0);
    f32x4 x[kSumHeads][PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int pos = min(span.position(place0 + 1024 * k), (span.len - 1) & ~3);
#pragma unroll
      for (int i = 0; i < kSumHeads; ++i)
        x[i][k] = *(const f32x4*)(scores + (int64_t)(pos & ~15) * a.G + (h0 + min(i, n - 1)) * 16 + (pos & 15));
    }
    if (h0 > 0) __syncthreads();
    if (wave < n) {
      const int hg = h0 + wave, hq = g * a.G + hg;
      f32x2 st = ((const f32x2*)((const char*)a.workspace + A.p.stats_at))[(int64_t)b * Hq + hq];
      if (A.p.workgroups > 0) {
        const int64_t mt = ((const int64_t*)((const char*)a.workspace + A.p.meta_at))[(int64_t)bg * A.p.head_tiles + hg / kPaHeads];
        const int first = (int)(uint32_t)mt, count = (int)(mt >> 32);
        if (count > 1)
          st = joined_stats((const f32x2*)((const char*)a.workspace + A.p.ml_at) + hg % kPaHeads, first, count,
                            a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf);
      }
      if (lane == 0) stats[wave] = f32x2{st[0], st[1] == 0.0f ? 0.0f : 1.0f / st[1]};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSumHeads; ++i) {
      if (i < n) {
        const f32x2 st = stats[i];
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[k][j] += exp2_fast(x[i][k][j] - st[0]) * st[1];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int pos = span.position(place0 + 1024 * k);
    if (all_seen(pos)) {
      *(f32x4*)(to + pos) = old[k] + f32x4{sum[k][0], sum[k][1], sum[k][2], sum[k][3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((pos + j >= span.lo || pos + j < span.first) && pos + j < span.len) to[pos + j] += sum[k][j];
    }
  }
}

// What is left to do behind the shares: blocks below `join_blocks` join, the others add up weights.
template <class M, int SPLIT, int PER>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const KernelArgs A, int padded, int groups,
                                                                   int join_blocks, int chunks) {
  __shared__ f32x4 lds[kPaWaves][64];
  if ((int)blockIdx.x < join_blocks)
    join_heads<M, SPLIT>(A, padded, groups, lds);
  else
    add_weights<PER>(A, blockIdx.x - join_blocks, chunks, (f32x2*)lds);
}

template <class M, int SPLIT>
void launch_join(const KernelArgs& A, int padded, hipStream_t stream) {
  const PagedAttentionArgs& a = A.a;
  const int heads = std::min(a.G, kPaHeads), groups = SPLIT > 1 ? heads : (heads + 3) / 4;
  const int join_blocks = A.p.workgroups > 0 ? (SPLIT > 1 ? A.p.items : A.p.workgroups) * groups : 0;
  const int seen = a.sums == nullptr ? 0 : most_seen(a.max_len, a.window, a.keep_first);
  // (four times the positions a block where the card has blocks enough, for fewer latencies in a row)
  const bool many = (int64_t)a.B * a.Hkv * ((seen + 1023) / 1024) > 2048;
  const int chunks = many ? (seen + 4095) / 4096 : (seen + 1023) / 1024;
  const int blocks = join_blocks + a.B * a.Hkv * chunks;
  if (blocks == 0) return;
  if (many)
    hipLaunchKernelGGL((paged_attention_join_kernel<M, SPLIT, 4>), dim3(blocks), dim3(256), 0, stream, A, padded, groups,
                       join_blocks, chunks);
  else
    hipLaunchKernelGGL((paged_attention_join_kernel<M, SPLIT, 1>), dim3(blocks), dim3(256), 0, stream, A, padded, groups,
                       join_blocks, chunks);
}

template <class M, bool FP8, int DP, bool SCALES>
void launch_width(const KernelArgs& A, hipStream_t stream) {
  const dim3 grid(A.p.workgroups > 0 ? A.p.workgroups : A.p.items), block(256);
  const bool aligned_pages = A.a.page_size % 16 == 0, full = A.a.D == DP;
  if (aligned_pages && full)
    hipLaunchKernelGGL((paged_attention_kernel<M, FP8, DP, true, true, SCALES>), grid, block, 0, stream, A);
  else if (aligned_pages)
    hipLaunchKernelGGL((paged_attention_kernel<M, FP8, DP, true, false, SCALES>), grid, block, 0, stream, A);
  else if (full)
    hipLaunchKernelGGL((paged_attention_kernel<M, FP8, DP, false, true, SCALES>), grid, block, 0, stream, A);
  else
    hipLaunchKernelGGL((paged_attention_kernel<M, FP8, DP, false, false, SCALES>), grid, block, 0, stream, A);
}

template <class M, bool FP8, bool SCALES>
void launch_kind(const KernelArgs& A, hipStream_t stream) {
  const int padded = pa_padded_width(A.a.D, FP8);
  switch (padded) {
    case 64: launch_width<M, FP8, 64, SCALES>(A, stream); break;
    case 96: if constexpr (!FP8) launch_width<M, FP8, 96, SCALES>(A, stream); break;
    case 128: launch_width<M, FP8, 128, SCALES>(A, stream); break;
    case 192: launch_width<M, FP8, 192, SCALES>(A, stream); break;
    default: launch_width<M, FP8, 256, SCALES>(A, stream); break;
  }
  if (A.p.workgroups >= 16 * A.p.items)
    launch_join<M, 4>(A, padded, stream);
  else
    launch_join<M, 1>(A, padded, stream);
}

}  // namespace

PagedAttentionPlan paged_attention_plan(int kind, int B, int Hkv, int G, int D, int max_len, int window,
                                        int keep_first, bool counted) {
  PagedAttentionPlan p{};
  p.head_tiles = (G + kPaHeads - 1) / kPaHeads;
  p.items = B * Hkv * p.head_tiles;
  const int seen = most_seen(max_len, window, keep_first);
  const int units = (seen + kPaUnit - 1) / kPaUnit;
  // Up to 8 units an item is one workgroup's and there is no second launch (64 heads on 8, 1000
  // positions: 1 sequence 10.0 us against 7.2 + 3.9, 8 sequences 11.0 / 8.6 + 4.0, 64 sequences
  // 21.3 / 21.9 + 4.3; 2000 positions: 15.4 / 6.2 + 4.0, 17.9 / 10.3 + 4.6, 35.8 / 30.2 + 4.7).
  // Shares of less than 2 units would leave more partial results than they save time.
  p.min_units = 2;
  const bool fp8 = kind >= kKvFp8Bf16;
  const int padded = pa_padded_width(D, fp8);
  p.workgroups = units > 8 ? 256 * residents(padded) : 0;
  // More than 16 query heads a key/value head: every tile of 16 has an equal part of the workgroups and
  // the same shares, and workgroups that read the same at about the same time sit on one XCD (8
  // workgroups apart), so that the cache comes from memory about once.  Tiles as items one behind the
  // other: 33 sequences of up to 14156 positions, 16 heads of 24: 393 us against 336 (1.08 GB; two tiles);
  // one of 131071, 2 heads of 48: 63 / 50; 255 on an 8-bit cache, 1 head of 64: 180 / 148; only with kept
  // scores, which go out twice as well, 998 / 1014.  Beyond 16 tiles a part would be a few workgroups.
  p.tile_groups = p.workgroups > 0 && p.head_tiles <= 16 ? p.head_tiles : 1;
  p.group_workgroups = p.tile_groups > 1 ? p.workgroups / p.tile_groups / 8 * 8 : p.workgroups;
  size_t at = 0;
  auto part = [&at](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
  if (p.workgroups > 0) {
    const size_t slots = 2 * (size_t)p.workgroups;
    p.ends_at = part((size_t)p.workgroups * 16);
    p.meta_at = part((size_t)p.items * 8);
    p.ml_at = part(slots * kPaHeads * 8);
    p.part_at = part(slots * kPaHeads * padded * 4);
  }
  if (counted) {
    p.stats_at = part((size_t)B * Hkv * G * 8);
    p.score_pitch = (max_len + 15) / 16 * 16;   // positions
    p.scores_at = part((size_t)B * Hkv * G * p.score_pitch * 4);
  }
  p.bytes = at;
  return p;
}

void launch_paged_attention(const PagedAttentionArgs& a, int kind, hipStream_t stream) {
  KernelArgs A{};
  A.a = a;
  A.p = paged_attention_plan(kind, a.B, a.Hkv, a.G, a.D, a.max_len, a.window, a.keep_first, a.sums != nullptr);
  A.by_page = fast_div(a.page_size);
  A.by_block = fast_div(a.scale_blocks > 0 ? a.page_size / a.scale_blocks : 1);
  const bool scales = a.scale_blocks > 0;
  switch (kind) {
    case kKvBf16: launch_kind<Bf16, false, false>(A, stream); break;
    case kKvF16: launch_kind<F16, false, false>(A, stream); break;
    case kKvFp8Bf16:
      if (scales) launch_kind<Bf16, true, true>(A, stream); else launch_kind<Bf16, true, false>(A, stream);
      break;
    default:
      if (scales) launch_kind<F16, true, true>(A, stream); else launch_kind<F16, true, false>(A, stream);
      break;
  }
}

}  // namespace vk

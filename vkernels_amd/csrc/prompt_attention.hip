// prompt_attention.hip — the attention of several new tokens of every sequence over a paged key-value cache.
//
// Token i of n new ones of a sequence of L positions is at p = L - n + i and sees positions j <= p, with a window w
// those with j > p - w or j < keep_first.  As for one token,
//   s_j = scale k_j q . k_j   (c tanh(s_j / c) with a softcap c),
//   out = sum_j e^{s_j} v_j / (sum_j e^{s_j} + e^{sink}),
// in one pass over keys and values with a running reference m of the exponents and their sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attention_math.hpp"
#include "fast_div.hpp"
#include "kv_rows.hpp"
#include "paged_attention.hpp"
#include "paged_attention_layout.hpp"
#include "prompt_attention.hpp"

namespace vk {
namespace {

using namespace attention;

constexpr float kFall = 14.0f;      // weights stay 2^7 above the smallest fp16 value that has all its bits
constexpr float kLeastScale = 0x1p-60f, kMostScale = 0x1p60f;      // of values, that fp16 weights follow
constexpr int kWaves = 4, kWaveRows = kPromptRows / kWaves;
static_assert(kWaveRows == 32, "a wavefront's rows are the columns of a matrix instruction");

struct KernelArgs {
  PromptAttentionArgs a;
  PromptAttentionPlan p;
  FastDiv by_page, by_block, by_group, by_heads, by_splits;
};

// What a workgroup works on.
struct Tile {
  int b;             // the sequence; B: behind the last one
  int slot, head, split;
  int s0, tokens;    // the sequence's first row of q, and how many it has
  int first, rows;   // its first row of the tile (negative: in front of the first sequence), and rows of the sequence
};
// False: the workgroup has no sequence's rows.
__device__ __forceinline__ bool find_tile(const KernelArgs& A, int block, Tile* t) {
  const PromptAttentionArgs& a = A.a;
  // Key/value heads in neighbouring workgroups, which different XCDs take: with 8 heads each XCD's cache has one
  // head's keys and values.  The last tiles of a sequence, which see most, come first.
  const int rest = divided(block, A.by_heads);
  t->head = block - rest * a.Hkv;
  const int from_end = divided(rest, A.by_splits);
  t->split = rest - from_end * A.p.splits;
  t->slot = A.p.slots - 1 - from_end;
  auto start = [&](int i) { return min(max(a.starts[i], 0), a.tokens); };
  // The tiles (of R rows) of sequence b begin at start rows / R + b: it has at most as many as lie up to the next one's.
  auto base = [&](int i) { return (start(i) * a.G >> A.p.row_shift) + i; };
  t->b = __builtin_amdgcn_readfirstlane(last_not_above(a.B + 1, t->slot, base));
  const int k = t->slot - base(t->b);
  t->s0 = start(t->b);
  t->tokens = (t->b < a.B ? max(start(t->b + 1), t->s0) : a.tokens) - t->s0;
  t->first = k << A.p.row_shift;
  t->rows = t->tokens * a.G;
  return k >= 0 && t->first < t->rows && t->b < a.B;
}

// Rows that belong to no sequence: those in front of the first one in the slots that lie there, what is left of them and
// those behind the last one in the slots behind it (there is one always).
__device__ __forceinline__ void clear_rows(const KernelArgs& A, const Tile& t) {
  const PromptAttentionArgs& a = A.a;
  if (!a.clear_rest || t.split > 0) return;
  const int pieces = a.D / 8;
  auto clear = [&](int begin, int end) {
    for (int i = threadIdx.x; i < (end - begin) * pieces; i += 256) {
      const int r = begin + i / pieces, tok = divided(r, A.by_group);
      const int64_t row = ((int64_t)tok * a.Hkv + t.head) * a.G + (r - tok * a.G);
      *(u32x4*)((char*)a.out + (row * a.D + i % pieces * 8) * 2) = u32x4{0, 0, 0, 0};
      if (i % pieces == 0 && a.lse != nullptr) a.lse[row] = kNegInf;
    }
  };
  if (t.first < 0) clear(t.slot << A.p.row_shift, (t.slot + 1) << A.p.row_shift);
  if (t.b < a.B) return;
  const int front = min(max(a.starts[0], 0), a.tokens) * a.G, begin = t.s0 * a.G + t.first, end = a.tokens * a.G;
  if (t.first == 0) clear(front & -(1 << A.p.row_shift), front);
  clear(begin, min(begin + (1 << A.p.row_shift), end));
}

// The positions a tile sees, as a line of places: the first `split` of them the positions at the beginning, the
// others positions `shift` further on.
struct Walk {
  int split, shift, tiles;
  __device__ __forceinline__ int position(int place) const { return place < split ? place : place + shift; }
};
// (hi: behind the last position that the tile's last row sees; lo: the first of its first row's window)
__device__ __forceinline__ Walk walk_of(int lo, int hi, int keep_first) {
  Walk w;
  const int first = min(keep_first, lo);
  w.split = (first + kPromptKeys - 1) & ~(kPromptKeys - 1);
  w.shift = (lo & ~15) - w.split;
  if (w.shift <= 0 && first > 0) w.split = w.shift = 0;
  w.tiles = hi <= 0 ? 0 : (hi - w.shift + kPromptKeys - 1) / kPromptKeys;
  return w;
}

template <int DP>
struct Layout {
  static constexpr int kLanes = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;   // threads that load a row: 8 values each
  static constexpr int kWaveLoad = 64 / kLanes;                // rows that a wavefront loads at once
  static constexpr int kPass = kWaves * kWaveLoad;             // ... and the workgroup
  static constexpr int kLoads = kPromptKeys / kPass;
  static constexpr int kPitch = kLanes * 16;                   // bytes of a row in LDS
  static constexpr int kTile = kPromptKeys * kPitch;
  static constexpr int kLds = 4 * kTile;                       // two buffers for keys, two for values
  // Where in its row a piece of 16 bytes lies: exchanged by the row (each exchange its own inverse), so that what is read at
  // once spreads over the banks: one piece of 16 rows (keys), two neighbouring pairs of pieces of 4 rows (values, by the
  // transposed reads).  No bank is asked for twice; with the pairs of two rows in one place a third of the cycles that
  // LDS was busy were conflicts, which the time did not show.
  static __device__ __forceinline__ int key_turn(int row) { return DP <= 64 ? (row >> 1) & 7 : row & 15; }
  static __device__ __forceinline__ int value_turn(int row) { return DP <= 64 ? row & 2 : (row & 3) * 2; }
  static __device__ __forceinline__ int key_piece(int slot, int row) { return slot ^ key_turn(row); }
  static __device__ __forceinline__ int value_piece(int slot, int row) { return slot ^ (value_turn(row) * 2); }
};

typedef __attribute__((address_space(3))) char* Lds;
typedef __attribute__((address_space(3))) u32x4* LdsPiece;
typedef __attribute__((address_space(3))) u32x2* LdsCodes;

// 16 bytes a lane from `from` to LDS, at `to` (uniform) + 16 lane.  Not waited for.
__device__ __forceinline__ void dma16(const char* from, Lds to) {
  const uint32_t at = (uint32_t)(uintptr_t)to;
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                   :
                   : "s"(__builtin_amdgcn_readfirstlane(at)), "v"(from)
                   : "memory");
}

// Is a 16-bit value (in the lower half of x) a finite number?
template <class W>
__device__ __forceinline__ bool finite(uint32_t x) {
  constexpr uint32_t kExponent = std::is_same_v<W, F16> ? 0x7C00u : 0x7F80u;
  return (x & kExponent) != kExponent;
}

// Zeros for what is no finite number among 8 values; whether there was one.  (An exponent of ones carries into
// the half's sign.)
template <class W>
__device__ __forceinline__ bool drop_others(u32x4& v) {
  constexpr uint32_t kExponents = std::is_same_v<W, F16> ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t kOnes = std::is_same_v<W, F16> ? 0x04000400u : 0x00800080u;
  uint32_t all = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t bad = ((v[e] & kExponents) + kOnes) & 0x80008000u;
    v[e] &= ~((bad >> 15) * 0xFFFFu);
    all |= bad;
  }
  return all != 0;
}

// The same among 16 E4M3 codes: 0x7F and 0xFF.
__device__ __forceinline__ bool drop_codes(u32x4& v) {
  uint32_t all = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t bad = ((v[e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    v[e] &= ~((bad >> 7) * 0xFFu);
    all |= bad;
  }
  return all != 0;
}

// The larger (the sum) of a value here and 32 lanes on.
__device__ __forceinline__ float over_halves_max(float x) {
  const u32x2 both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float over_halves_sum(float x) {
  const u32x2 both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// Bits below n of 32.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

// Brings the reference m of a row's weights to its largest new score where that passes it by kSlack; the sums are
// relative to it.  (A row by itself: what it gives does not depend on the rows beside it; of an 8-bit cache, where a tile that
// all rows see is looked at by its largest score and scale, within rounding.)
// FALLS: down as well, where all new scores are more than kFall below.  Weights in fp16 end at 2^-24, and positions far below
// one of large weight may be the whole result, where that one's value is small.  The sums take steps of up to 2^40 until
// the weights' reaches 2^40: so they stay in range times any value.  What is still lost is 2^-18 of the largest weight among
// a weight's own 32 positions (2^-7 or more in fp16, a half step at most 2^-25), and what is below 2^-60 of the row's.
// PEAK: the weighted sums are not bound by the weights' (their scales are on top), and the reference stays within 2^60 of its
// highest place.
template <bool FALLS, bool PEAK, int N>
__device__ __forceinline__ void follow(float top, float& m, float& l, f32x16 (&acc)[N], float& peak) {
  // (one comparison for both sides)
  const float middle = (kSlack - kFall) / 2;
  if (!__any(FALLS ? fabsf(top - m - middle) > kSlack - middle : top > m + kSlack)) return;
  float m_new = top > m + kSlack ? top : m;
  if constexpr (FALLS) {
    if (over_halves_max(l) < 0x1p40f && top < m - kFall && top > kNegInf && (!PEAK || m > peak - 20.0f)) m_new = fmaxf(top, m - 40.0f);
  }
  if constexpr (PEAK) peak = fmaxf(peak, m_new);
  const float fix = exp2_fast(m - or_zero(m_new));
  m = m_new;
  l *= fix;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] *= fix;
}

// S^T = K q^T and O^T += V^T P^T, both 32 x 32 x 16 with the keys (the head's width) as rows and a wavefront's 32
// rows as columns: a lane holds half of one row's scores, so that maximum, sum and rescaling stay in the lane and its
// neighbour 32 lanes on, and its weights are where the second product wants them, in the order of positions in
// which the values are read from LDS (transposed, 4 x 16 at a time).
// Keys and values of 64 positions go to LDS without a register between (8-bit ones through registers, where they
// become 16-bit ones), a tile ahead, in two buffers each.  A wavefront takes 32 positions at a time and works out
// the scores of the next 32 beside the weights of these, so that the matrix instructions run under the exponentials: the
// tiles of keys are 32 positions on from those of values, and both are done with when a tile ends.
// 4096 tokens over 16384 positions, 32 heads on 8 of 128: 1.02 ms, 945 TFLOP/s (a bf16 product of 8192^3 reaches 1379);
// heads of 64: 1.19 ms for as many products, 810.  Matrix instructions take 45 % of the cycles, vector ones 53 %; without
// the loads it is 0.89 ms, without the exponentials 1.05: these are hidden, loads are an eighth, and what keeps the
// rest above the products' 0.70 is not known.  Keys and values through registers, no scores ahead: 1.21;
// scores ahead in the compiler's own order: 1.24 (every read from LDS waited for), 1.08 by its scheduling groups.
// Two chains of scores, reads 2 or 5 operands ahead, and priorities for either half change nothing or cost 2 %.
template <class M, bool FP8, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void prompt_attention_kernel(const KernelArgs A) {
  typedef Layout<DP> L;
  // What values and weights are multiplied in.  Codes are exact in fp16, and weights times the values' scales have three bits
  // more there than in bf16, whose errors would be larger than the result's own rounding (2.5e-3 against 1.7e-3 in bf16
  // results, where fp16 weights leave 1.7e-3; 1.42 against 1.23 ms).  fp16 does not have every scale's range, so that the
  // reference of the weights follows weight times scale; rows that see scales outside 2^-60 .. 2^60 are worked on again.
  typedef std::conditional_t<FP8, F16, M> W;
  const PromptAttentionArgs& a = A.a;
  __shared__ __attribute__((aligned(16))) char lds[L::kLds];
  __shared__ __attribute__((aligned(16))) float scale_lds[FP8 ? kWaves : 1][3][2 * kPromptKeys];   // as well
  __shared__ int64_t row_lds[kWaves][2 * kPromptKeys];      // by the place mod 128
  __shared__ uint32_t any_bad;      // values that are no finite numbers have been left out

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile t;
  const int Hq = a.Hkv * a.G;
  if (!find_tile(A, blockIdx.x, &t)) {
    clear_rows(A, t);
    return;
  }

  const int len = min(max(a.lens[t.b], 0), a.max_len), before = len - t.tokens;
  // this lane's row, and the positions of the wavefront's and the workgroup's first and last rows
  const int wave_first = t.first + wave * kWaveRows;
  const bool valid = wave_first + n < t.rows;
  const int row = min(wave_first + n, t.rows - 1), tok = divided(row, A.by_group), g = row - tok * a.G;
  const int place = before + tok;
  const int wave_lo = before + divided(min(wave_first, t.rows - 1), A.by_group);
  const int wave_hi = before + divided(min(wave_first + kWaveRows, t.rows) - 1, A.by_group);
  const int tile_lo = before + divided(t.first, A.by_group);
  const int tile_hi = before + divided(min(t.first + kPromptRows, t.rows) - 1, A.by_group);
  // positions up to `low` of a row's place are behind its window
  auto low_of = [&](int place) { return a.window > 0 ? max(place, a.window - 1) - a.window : -1; };
  const int low = low_of(place), wave_low = low_of(wave_lo);
  const int hi = tile_hi + 1;
  const Walk walk = walk_of(low_of(tile_lo) + 1, hi, a.keep_first);
  const int tile_begin = t.split * A.p.share, tile_end = min(walk.tiles, tile_begin + A.p.share);

  // Queries: the second operand of the first product.
  typename M::V8 q[DP / 16];
  {
    const char* const from = (const char*)a.q + ((int64_t)(t.s0 + tok) * a.q_stride_t + (int64_t)(t.head * a.G + g) * a.q_stride_h) * 2;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int d = i * 16 + half * 8;
      const u32x4 x = *(const u32x4*)(from + (d < a.D ? d : 0) * 2);
      q[i] = as_v8<M>(d < a.D ? x : u32x4{0, 0, 0, 0});
    }
  }
  const float k_scale = FP8 ? 1.0f : a.scale;      // (8-bit keys: with the positions' scales)
  const bool plain = !(a.softcap > 0.0f) && (FP8 || a.scale > 0.0f);
  const float to_log2 = k_scale * kLog2e;
  const float cap_in = a.softcap > 0.0f ? 2.0f * k_scale * kLog2e / a.softcap : 0.0f, cap_out = a.softcap * kLog2e;

  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
  float m = kNegInf, l = 0.0f, peak = kNegInf;
  // (fp16 weights end at 2^-24: they are kept 2^7 above the reference, so that with the slack they reach 2^15)
  constexpr float kLift = std::is_same_v<W, F16> ? 7.0f : 0.0f;

  const int32_t* const table = a.table + (int64_t)t.b * a.table_stride;
  const int last_entry = divided(max(hi - 1, 0), A.by_page);
  constexpr int kElem = FP8 ? 1 : 2;
  const char* const kbase = (const char*)a.k_cache + (int64_t)t.head * a.head_stride * kElem;
  const char* const vbase = (const char*)a.v_cache + (int64_t)t.head * a.head_stride * kElem;
  const int64_t page_bytes = a.page_stride * kElem, slot_bytes = a.slot_stride * kElem;
  const int slot = tid % L::kLanes, slot_row = tid / L::kLanes;    // what this thread loads of a row, and of which rows
  auto lds_keys = [&](int tile) { return (Lds)&lds[0] + (tile & 1) * L::kTile; };
  auto lds_values = [&](int tile) { return (Lds)&lds[0] + (2 + (tile & 1)) * L::kTile; };
  // What lies behind a key's last value is zeros, once for all.
  if (a.D < DP) {
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      const int r = slot_row + i * L::kPass;
      if (L::key_piece(slot, r) * 8 >= a.D) {
        *(LdsPiece)(lds_keys(0) + r * L::kPitch + slot * 16) = u32x4{0, 0, 0, 0};
        *(LdsPiece)(lds_keys(1) + r * L::kPitch + slot * 16) = u32x4{0, 0, 0, 0};
      }
    }
  }

  // The table's entry for a place of a tile of keys (which begin half a tile behind the tile's beginning), a lane each,
  // asked for a tile ahead.
  auto ask = [&](int tile) {
    const int pos = walk.position(max(tile * kPromptKeys + kPromptKeys / 2 + lane, 0));
    return table[min(divided(pos, A.by_page), last_entry)];
  };
  u32x2 kreg[L::kLoads], vreg[L::kLoads];      // (8-bit caches)
  float ks = 1.0f, vs = 1.0f;
  // The largest value scale (in powers of two) of the 32 positions behind an even sub, behind an odd one.
  float range_of[2] = {0.0f, 0.0f};
  // A lane works out where its place's rows lie, for the wavefront's lanes that load them; which of the places there are.
  auto find_rows = [&](int tile, int entry) -> uint64_t {
    const int at_place = tile * kPromptKeys + kPromptKeys / 2 + lane, pos = walk.position(max(at_place, 0));
    const int ids = at_place >= 0 && pos < hi && (uint32_t)entry < (uint32_t)a.num_pages ? entry : -1;
    const int in_page = pos - divided(pos, A.by_page) * a.page_size;
    row_lds[wave][at_place & (2 * kPromptKeys - 1)] = max(ids, 0) * page_bytes + (uint32_t)in_page * (uint64_t)(uint32_t)slot_bytes;
    if constexpr (FP8) {
      const int64_t at = a.scale_blocks == 0 ? t.head
                                             : ((int64_t)max(ids, 0) * a.Hkv + t.head) * a.scale_blocks + divided(in_page, A.by_block);
      ks = ids >= 0 ? a.k_scale[at] * a.scale : 0.0f;
      vs = ids >= 0 ? a.v_scale[at] : 0.0f;
    }
    // (lanes read what other lanes of their wavefront wrote: LDS keeps the order, and so must the compiler)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return __ballot(ids >= 0);
  };
  auto load = [&](int tile, const char* base, bool values, u32x2* regs) {
    const Lds to = values ? lds_values(tile) : lds_keys(tile);
    const int place0 = tile * kPromptKeys + (values ? 0 : kPromptKeys / 2);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      const int r = slot_row + i * L::kPass, piece = values ? L::value_piece(slot, r) : L::key_piece(slot, r);
      const char* const from = base + row_lds[wave][(place0 + r) & (2 * kPromptKeys - 1)];
      if constexpr (FP8) {
        regs[i] = *(const u32x2*)(from + (piece * 8 < a.D ? piece * 8 : 0));
      } else {
        if (piece * 8 < a.D) dma16(from + piece * 16, to + (i * L::kPass + wave * L::kWaveLoad) * L::kPitch);
      }
    }
  };
  auto load_keys = [&](int tile) { load(tile, kbase, false, kreg); };
  auto load_values = [&](int tile) { load(tile, vbase, true, vreg); };
  // Does any row of the workgroup not see all of a tile?
  auto partial = [&](int pos0) {
    return pos0 + kPromptKeys - 1 > tile_lo ||
           (a.window > 0 && pos0 <= low_of(tile_hi) && pos0 + kPromptKeys > a.keep_first);
  };
  // Values as the product may have them: positions that there are not as zeros, and where some rows do not see all of
  // the tile, values that are no finite numbers as well: a weight of 0 times them would not be 0 (they are added in
  // the end).
  auto clean = [&](u32x4 v, bool there, bool look) {
    if (!there) v = u32x4{0, 0, 0, 0};
    if (look && drop_others<W>(v)) any_bad = 1;
    return v;
  };
  // 8-bit keys and values out of the registers, and their scales.
  auto put_keys = [&](int tile) {
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      const int r = slot_row + i * L::kPass;
      union { typename M::V8 v; u32x4 u; } k;
      k.v = fp8x8<M>(kreg[i][0], kreg[i][1]);
      if (L::key_piece(slot, r) * 8 < a.D) *(LdsPiece)(lds_keys(tile) + r * L::kPitch + slot * 16) = k.u;
    }
    const int at = (tile * kPromptKeys + kPromptKeys / 2 + lane) & (2 * kPromptKeys - 1);
    scale_lds[wave][0][at] = ks;
    scale_lds[wave][1][at] = vs;
    // (From 2^-60, 0 among them, to 2^60: a step of the reference from one end to the other stays within 32 bits, so that
    // the sum of weights keeps positions whose values are 0.  A scale that is not seen may be anything.)
    float range = fminf(fmaxf(__builtin_amdgcn_logf(fabsf(vs)), -60.0f), 60.0f);
    scale_lds[wave][2][at] = range;
    // (the largest of 16 lanes by rotations within them)
    auto with = [&](float other) { range = fmaxf(range, other); };
    with(__uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(range), 0x128, 0xF, 0xF, false)));
    with(__uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(range), 0x124, 0xF, 0xF, false)));
    with(__uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(range), 0x122, 0xF, 0xF, false)));
    with(__uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(range), 0x121, 0xF, 0xF, false)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float most = fmaxf(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(range), i * 32)),
                               __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(range), i * 32 + 16)));
      range_of[i] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(most)));
    }
  };
  auto put_values = [&](int tile, uint64_t there) {
    const bool look = partial(walk.position(tile * kPromptKeys));
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      const int r = slot_row + i * L::kPass;
      union { typename W::V8 v; u32x4 u; } v;
      v.v = fp8x8<W>(vreg[i][0], vreg[i][1]);
      if (L::value_piece(slot, r) * 8 < a.D)
        *(LdsPiece)(lds_values(tile) + r * L::kPitch + slot * 16) = clean(v.u, (there >> r) & 1, look);
    }
  };
  // 16-bit values that are in LDS already.
  auto clean_values = [&](int tile, uint64_t there, bool look) {
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      const int r = slot_row + i * L::kPass;
      const LdsPiece at = (LdsPiece)(lds_values(tile) + r * L::kPitch + slot * 16);
      if (L::value_piece(slot, r) * 8 < a.D) *at = clean(*at, (there >> r) & 1, look);
    }
  };
  auto landed = [&] {
    if constexpr (!FP8) __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // Hidden from every row of the wavefront: behind the last one's place, or in front of the first one's window.
  constexpr int kSub = kPromptKeys / 2;
  auto hidden = [&](int sub) {
    const int pos0 = walk.position(sub * kSub);
    return pos0 > wave_hi || (pos0 + kSub - 1 <= wave_low && pos0 >= a.keep_first) || wave_first >= t.rows;
  };
  const int key_at = n * L::kPitch + (half ^ L::key_turn(n)) * 16;
  // Scores of 32 positions: sub - 1 of its tile of keys.
  auto read_keys = [&](int sub, int i) {
    const Lds keys = lds_keys((sub - 1) >> 1) + ((sub - 1) & 1) * kSub * L::kPitch;
    return as_v8<M>(*(LdsPiece)(keys + (key_at ^ (i * 32))));
  };
  f32x16 zero;
#pragma unroll
  for (int j = 0; j < 16; ++j) zero[j] = 0.0f;
  // The scales of the keys (values) that four of a lane's scores belong to.
  auto scales_of = [&](int sub, int values, int j) {
    return *(const f32x4*)&scale_lds[wave][values][(sub * kSub & (2 * kPromptKeys - 1)) + j * 2 + half * 4];
  };
  auto score = [&](int sub, f32x16& s) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) s = M::mfma(read_keys(sub, i), q[i], i == 0 ? zero : s);
    if constexpr (FP8) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const f32x4 f = scales_of(sub, 0, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j + i] *= f[i];
      }
    }
  };
  const int quarter = (lane >> 4) & 1, l16 = lane & 15;
  const int value_row = half * 4 + (l16 >> 2), value_turn = L::value_turn(value_row);
  const int value_at = value_row * L::kPitch + (l16 & 3) * 8;
  // Positions 16 j .. 16 j + 15 of a sub, 32 of the head's values; and all of those times their weights.
  auto read_values = [&](int sub, int j, int i) {
    const Lds column = lds_values(sub >> 1) + ((sub & 1) * kSub + j * 16) * L::kPitch + value_at +
                               ((i * 2 + quarter) ^ value_turn) * 32;
    union { i16x4 h[2]; typename W::V8 v; } v;
    v.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)column);
    v.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(column + 8 * L::kPitch));
    return v.v;
  };
  auto add_values = [&](int sub, int j, typename W::V8 p) {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = W::mfma(read_values(sub, j, i), p, acc[i]);
  };
  // What the reference follows of a sub's scores, c times which is in powers of two: the largest (of both halves).
  auto largest = [&](int sub, const f32x16& x, float c) {
    if constexpr (FP8) {
      float top = kNegInf;
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const f32x4 f = scales_of(sub, 2, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fmaf(x[j + i], c, f[i]));
      }
      return over_halves_max(top);
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, x[j]);
    return over_halves_max(top) * c;
  };
  auto follow_scores = [&](float top) { follow<std::is_same_v<W, F16>, FP8>(top, m, l, acc, peak); };

  // The same where every row of the workgroup sees all of the sub and the scores need nothing but their factor: one
  // stretch of code in a fixed order, reads from LDS three operands ahead and the exponentials (then the next
  // scores' maximum) between the matrix instructions.  `top`: what the reference follows, of the next sub afterwards.
  auto attend_whole = [&](int sub, const f32x16& x, f32x16& next, float& top) {
    constexpr int kSteps = DP / 16, kAhead = 3;
    follow_scores(top);
    const float ref = or_zero(m) - kLift;
    union { typename W::T e[16]; typename W::V8 v[2]; } p;
    typename M::V8 k[kSteps];
    typename W::V8 v[kSteps];
    f32x4 f;                     // (8-bit caches: scales)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) k[i] = read_keys(sub + 1, i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      next = M::mfma(k[i], q[i], i == 0 ? zero : next);
      if (i + kAhead < kSteps)
        k[i + kAhead] = read_keys(sub + 1, i + kAhead);
      else
        v[i + kAhead - kSteps] = read_values(sub, (i + kAhead - kSteps) / (DP / 32), (i + kAhead - kSteps) % (DP / 32));
#pragma unroll
      for (int j = 16 * i / kSteps; j < 16 * (i + 1) / kSteps; ++j) {
        const float w = exp2_fast(__builtin_fmaf(x[j], to_log2, -ref));
        l += w;
        if constexpr (FP8) {
          if (j % 4 == 0) f = scales_of(sub, 1, j);
          p.e[j] = (typename W::T)(w * f[j % 4]);
        } else {
          p.e[j] = (typename W::T)w;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    float most[2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      acc[i % (DP / 32)] = W::mfma(v[i], p.v[i / (DP / 32)], acc[i % (DP / 32)]);
      if (i + kAhead < kSteps) v[i + kAhead] = read_values(sub, (i + kAhead) / (DP / 32), (i + kAhead) % (DP / 32));
#pragma unroll
      for (int j = 16 * i / kSteps; j < 16 * (i + 1) / kSteps; ++j) {
        if constexpr (FP8) {
          if (j % 4 == 0) f = scales_of(sub + 1, 0, j);
          next[j] *= f[j % 4];
        }
        most[j & 1] = j < 2 ? next[j] : fmaxf(most[j & 1], next[j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    top = __builtin_fmaf(over_halves_max(fmaxf(most[0], most[1])), to_log2, FP8 ? range_of[sub & 1] : 0.0f);
  };

  // Positions of a sub, whose scores are in `x`, and the scores of the next one (skip_next: not those).
  auto attend = [&](int sub, uint32_t there, f32x16& x, f32x16& next, bool skip_next) {
    const int pos0 = walk.position(sub * kSub);
    const bool whole = there == ~0u && pos0 + kSub - 1 <= wave_lo &&
                       (a.window <= 0 || pos0 > low_of(wave_hi) || pos0 + kSub <= a.keep_first);
    if (!skip_next) score(sub + 1, next);
    if (hidden(sub)) return;
    // Scores in powers of two, unless they are taken there with the reference.
    float c = to_log2;
    if (!plain) {
      c = 1.0f;
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = capped(x[j] * cap_in, cap_out);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= to_log2;
      }
    }
    uint32_t sees = ~0u;      // the positions that this lane's row sees
    if (!whole) {
      sees = bits_below(place + 1 - pos0) & (~bits_below(low + 1 - pos0) | bits_below(a.keep_first - pos0)) & there;
      sees >>= half * 4;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (!((sees >> (j / 4 * 8 + j % 4)) & 1)) x[j] = kNegInf;
      }
    }
    follow_scores(largest(sub, x, c));
    const float ref = or_zero(m) - kLift;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      union { typename W::T e[8]; typename W::V8 v; } p;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        f32x4 f = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (FP8) f = scales_of(sub, 1, g * 8 + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = g * 8 + i + e;
          const float w = exp2_fast(__builtin_fmaf(x[j], c, -ref));
          l += w;
          // (a scale that is not seen may be anything)
          p.e[i + e] = (typename W::T)(!FP8 ? w : whole || ((sees >> (j / 4 * 8 + j % 4)) & 1) ? w * f[e] : 0.0f);
        }
      }
      add_values(sub, g, p.v);
    }
  };

  if (tid == 0) any_bad = 0;
  if (tile_begin < tile_end) {
    // Which of a tile's positions there are: its second half and the next tile's first come with its keys.
    uint64_t there = find_rows(tile_begin - 1, ask(tile_begin - 1));
    load_keys(tile_begin - 1);
    if constexpr (FP8) {
      __syncthreads();      // (the zeros behind the keys)
      put_keys(tile_begin - 1);
    }
    uint32_t first = (uint32_t)(there >> 32);
    there = find_rows(tile_begin, ask(tile_begin));
    load_keys(tile_begin);
    load_values(tile_begin);
    int ids = ask(tile_begin + 1);
    landed();             // (any_bad as well)
    if constexpr (FP8) {
      put_keys(tile_begin);
      put_values(tile_begin, there << 32 | first);
      __syncthreads();
    }
    f32x16 even, odd;
    if (!hidden(2 * tile_begin)) score(2 * tile_begin, even);
    __syncthreads();
    uint64_t these = there << 32 | first;
    // The next tile's keys and values are on their way while this one's are multiplied.
    auto ahead = [&](int tile) {
      first = (uint32_t)(there >> 32);
      if (tile + 1 < tile_end) {
        there = find_rows(tile + 1, ids);
        load_keys(tile + 1);
        load_values(tile + 1);
        ids = ask(tile + 2);
      }
    };
    for (int tile = tile_begin; tile < tile_end;) {
      if (plain) {
        float top = largest(2 * tile, even, to_log2);
        for (; tile + 1 < tile_end && these == ~0ull && !partial(walk.position(tile * kPromptKeys)) && !hidden(2 * tile + 2); ++tile) {
          ahead(tile);
          attend_whole(2 * tile, even, odd, top);
          attend_whole(2 * tile + 1, odd, even, top);
          if constexpr (FP8) {
            put_keys(tile + 1);
            put_values(tile + 1, there << 32 | first);
          }
          landed();
          these = there << 32 | first;
        }
      }
      ahead(tile);
      const bool more = tile + 1 < tile_end;
      if constexpr (!FP8) {
        const bool look = partial(walk.position(tile * kPromptKeys));
        if (look || these != ~0ull) {
          clean_values(tile, these, look);
          __syncthreads();
        }
      }
      attend(2 * tile, (uint32_t)these, even, odd, hidden(2 * tile + 1));
      attend(2 * tile + 1, (uint32_t)(these >> 32), odd, even, !more || hidden(2 * tile + 2));
      if constexpr (FP8) {
        if (more) {
          put_keys(tile + 1);
          put_values(tile + 1, there << 32 | first);
        }
      }
      landed();
      these = there << 32 | first;
      ++tile;
    }
  }

  // What was left out is added to the row's sums in memory (the values that this lane has written): values at positions
  // that the row sees, whatever their weight.  An infinity stays one, or becomes NaN.
  auto add_bad = [&](auto* sums) {
#pragma unroll 1
    for (int tile = tile_begin; tile < tile_end; ++tile) {
      const int pos0 = walk.position(tile * kPromptKeys);
      if (!partial(pos0)) continue;
#pragma unroll 1
      for (int pos = pos0; pos < min(pos0 + kPromptKeys, hi); ++pos) {
        const int entry = divided(pos, A.by_page), id = table[entry];
        if (!(pos <= place && (pos > low || pos < a.keep_first)) || (uint32_t)id >= (uint32_t)a.num_pages) continue;
        const char* const from = vbase + (int64_t)id * page_bytes + (int64_t)(pos - entry * a.page_size) * slot_bytes;
#pragma unroll 1
        for (int d = half * 4; d < a.D; d += d % 4 == 3 ? 5 : 1) {
          union { uint16_t u; typename W::T t; } v;
          if constexpr (FP8)
            v.t = fp8x8<W>(((const uint8_t*)from)[d], 0)[0];
          else
            v.u = ((const uint16_t*)from)[d];
          if (!finite<W>(v.u)) sums[d] = (std::remove_reference_t<decltype(*sums)>)((float)sums[d] + (float)v.t);
        }
      }
    }
  };

  l = over_halves_sum(l);
  const float ref = or_zero(m) - kLift;        // l and the sums are relative to 2^ref
  if (A.p.splits > 1) {
    const int64_t slot = ((int64_t)t.slot * a.Hkv + t.head) * A.p.splits + t.split;
    const int at = wave * kWaveRows + n;
    if (half == 0) ((f32x2*)((char*)a.workspace + A.p.ml_at))[slot * kPromptRows + at] = f32x2{l == 0.0f ? kNegInf : ref, l};
    if (!valid || __all(l == 0.0f)) return;
    float* const part = (float*)((char*)a.workspace + A.p.part_at) + (slot * kPromptRows + at) * DP + half * 4;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(f32x4*)(part + i * 32 + j * 8) = f32x4{acc[i][j * 4], acc[i][j * 4 + 1], acc[i][j * 4 + 2], acc[i][j * 4 + 3]};
    if (any_bad && tile_begin < tile_end) add_bad(part - half * 4);
    return;
  }
  if (!valid) return;
  const int hq = t.head * a.G + g;
  const float sink = a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf;
  const float top = or_zero(fmaxf(l == 0.0f ? kNegInf : ref, sink));
  const float fix = l == 0.0f ? 0.0f : exp2_fast(ref - top);
  const float total = l * fix + exp2_fast(sink - top);
  const float inv = total == 0.0f ? 0.0f : fix / total;
  const int64_t out_row = (int64_t)(t.s0 + tok) * Hq + hq;
  if (a.lse != nullptr && half == 0) a.lse[out_row] = log_of_sum(top, total, a.sinks != nullptr ? a.sinks + hq : nullptr);
  char* const to = (char*)a.out + (out_row * a.D + half * 4) * 2;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      union { typename M::T e[4]; u32x2 u; } r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r.e[e] = (typename M::T)(acc[i][j * 4 + e] * inv);
      if (i * 32 + j * 8 + half * 4 < a.D) *(u32x2*)(to + (i * 32 + j * 8) * 2) = r.u;
    }
  }
  if (any_bad && tile_begin < tile_end) add_bad((typename M::T*)a.out + out_row * a.D);
}

// Does a row of the tile see a position whose value scale is outside of what fp16 weights follow?  (An infinite one or
// NaN makes the row what it is either way.)
__device__ __forceinline__ bool sees_far_scales(const KernelArgs& A, const Tile& t) {
  const PromptAttentionArgs& a = A.a;
  __shared__ uint32_t any_far;
  if (threadIdx.x == 0) any_far = 0;
  __syncthreads();
  const int before = min(max(a.lens[t.b], 0), a.max_len) - t.tokens;
  const int hi = before + divided(min(t.first + kPromptRows, t.rows) - 1, A.by_group) + 1;
  const int begin = a.window > 0 ? max(before + divided(t.first, A.by_group), a.window - 1) - a.window + 1 : 0;
  bool far = false;
  auto look = [&](float scale) {
    const float size = fabsf(scale);
    far |= size != 0.0f && (size < kLeastScale || size > kMostScale) && size < __builtin_inff();
  };
  if (a.scale_blocks == 0) {
    look(a.v_scale[t.head]);
  } else if (hi > 0) {
    // The blocks of the first positions, then those of the window (all, without one).
    const int32_t* const table = a.table + (int64_t)t.b * a.table_stride;
    const int block = a.page_size / a.scale_blocks, lo = divided(begin, A.by_block);
    const int first = a.keep_first > 0 ? min(lo, divided(a.keep_first - 1, A.by_block) + 1) : 0;
    const int blocks = first + divided(hi - 1, A.by_block) + 1 - lo;
    // (8 at a time, all of them loaded: the last one again behind it, an entry's that is no page from page 0)
    constexpr int kAtOnce = 8;
    for (int i0 = threadIdx.x; i0 < blocks; i0 += 256 * kAtOnce) {
      int id[kAtOnce], in_page[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int i = min(i0 + 256 * j, blocks - 1), pos = (i < first ? i : lo + i - first) * block;
        const int in_table = divided(pos, A.by_page);
        id[j] = table[in_table];
        in_page[j] = divided(pos - in_table * a.page_size, A.by_block);
      }
      float scale[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const bool there = (uint32_t)id[j] < (uint32_t)a.num_pages;
        scale[j] = a.v_scale[((int64_t)(there ? id[j] : 0) * a.Hkv + t.head) * a.scale_blocks + in_page[j]];
        if (!there) scale[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) look(scale[j]);
    }
  }
  if (__any(far)) any_far = 1;
  __syncthreads();
  return any_far != 0;
}

// A wavefront's 32 positions in LDS: rows as they are in the cache, pieces of 16 bytes exchanged by the row (each exchange
// its own inverse) so that 16 rows' pieces spread over the banks.
template <bool FP8, int DP>
struct FewLayout {
  typedef Layout<DP> L;
  static constexpr int kPitch = FP8 ? L::kPitch / 2 : L::kPitch, kLanes = kPitch / 16;
  static constexpr int kRows = 64 / kLanes, kLoads = 32 / kRows;      // rows that a load takes; loads
  // Straight to LDS, in two buffers, where two workgroups of those fit a CU; else by way of registers and one buffer
  // (32 sequences of up to 8192, 8 heads of 128 in bf16: 163 us with one workgroup a CU, 138 so).
  static constexpr bool kDirect = FP8 || DP <= 64;
  static constexpr int kBuffers = kDirect ? 2 : 1;
  static __device__ __forceinline__ int code_turn(int row) {
    return kLanes == 4 ? (row >> 2) & 3 : kLanes == 8 ? (row >> 1) & 7 : row & 15;
  }
  static __device__ __forceinline__ int key_piece(int slot, int row) {
    return FP8 ? slot ^ code_turn(row) : L::key_piece(slot, row);
  }
  // (codes of values are read two neighbouring pieces of rows 0 .. 3 and 8 .. 11, or 4 .. 7 and 12 .. 15, at once)
  static __device__ __forceinline__ int value_code_turn(int row) {
    return kLanes == 4 ? (row >> 3 & 1) * 2 : kLanes == 8 ? (row >> 1 & 1) * 2 + (row >> 3 & 1) * 4 : (row & 3) * 2 + (row >> 3 & 1) * 8;
  }
  static __device__ __forceinline__ int value_piece(int slot, int row) {
    return FP8 ? slot ^ value_code_turn(row) : L::value_piece(slot, row);
  }
  static __device__ __forceinline__ int value_pair(int pair, int row) { return pair ^ L::value_turn(row); }
};

// The same for tiles of 32 rows: every wavefront has all of the rows and takes every fourth 32 positions, by itself.  Keys
// and values go to the wavefront's own part of LDS as they are (8-bit codes become 16-bit values as they are read from
// there), the next ones on their way while these are multiplied.  The wavefronts' results meet in LDS at the end, one
// after the other.  Bound by latency: 5 tokens of 32 sequences of 1024 to 8192, 32 heads on 8 of 128 in 8 bits, 279 MB:
// 95 us (2.9 TB/s) of which a workgroup's start, six dependent loads, and end are a third; one sequence of 131071: 68
// (4.0 TB/s), in bf16 115 (4.7).  With tiles of 128 rows, one wavefront with all of them: 250.
// AGAIN: behind tiles of 128 rows over an 8-bit cache, the rows that see a value scale outside of what the fp16 weights
// there take (two bf16 terms take any), 32 of a tile's 128 after the other; without such a scale a workgroup only looks: 9 us
// for 4096 tokens over 16384 positions in blocks of 16, 36 where every position has its scale, beside 1.43 ms.
template <class M, bool FP8, int DP, bool AGAIN>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void prompt_attention_few_kernel(const KernelArgs A) {
  typedef std::conditional_t<FP8, Bf16, M> W;
  typedef FewLayout<FP8, DP> F;
  constexpr int kSub = 32, kSumPitch = DP + 4;
  const PromptAttentionArgs& a = A.a;
  union Shared {
    char tiles[kWaves][F::kBuffers][2][kSub * F::kPitch];   // keys and values
    float sums[kPromptFewRows][kSumPitch];        // (when all are done with those)
  };
  __shared__ __attribute__((aligned(16))) Shared lds;
  auto& sums = lds.sums;
  __shared__ __attribute__((aligned(16))) float scale_lds[FP8 ? kWaves : 1][2 * kSub];
  __shared__ int64_t row_lds[kWaves][kSub];
  __shared__ f32x2 ml_lds[kWaves][kPromptFewRows];

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile t;
  if (!find_tile(A, blockIdx.x, &t)) {
    if constexpr (!AGAIN) clear_rows(A, t);
    return;
  }
  if (AGAIN && !sees_far_scales(A, t)) return;
  const int last_row = min(t.first + kPromptRows, t.rows);      // (AGAIN)
  do {
    const int len = min(max(a.lens[t.b], 0), a.max_len), before = len - t.tokens;
    const int row = min(t.first + n, t.rows - 1), tok = divided(row, A.by_group), g = row - tok * a.G;
    const int place = before + tok;
    const int tile_lo = before + divided(t.first, A.by_group);
    const int tile_hi = before + divided(min(t.first + kPromptFewRows, t.rows) - 1, A.by_group);
    auto low_of = [&](int place) { return a.window > 0 ? max(place, a.window - 1) - a.window : -1; };
    const int low = low_of(place), hi = tile_hi + 1;
    const Walk walk = walk_of(low_of(tile_lo) + 1, hi, a.keep_first);
    const int subs = hi <= 0 ? 0 : (hi - walk.shift + kSub - 1) / kSub;
    const int sub_begin = t.split * A.p.share * 2, sub_end = min(subs, sub_begin + A.p.share * 2);
    if (sub_begin >= sub_end && A.p.splits > 1) {
      // (a shorter sequence's)
      const int64_t part = ((int64_t)t.slot * a.Hkv + t.head) * A.p.splits + t.split;
      if (tid < kPromptFewRows) ((f32x2*)((char*)a.workspace + A.p.ml_at))[part * kPromptFewRows + tid] = f32x2{kNegInf, 0.0f};
      return;
    }

    typename M::V8 q[DP / 16];
    {
      const char* const from = (const char*)a.q + ((int64_t)(t.s0 + tok) * a.q_stride_t + (int64_t)(t.head * a.G + g) * a.q_stride_h) * 2;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const int d = i * 16 + half * 8;
        const u32x4 x = *(const u32x4*)(from + (d < a.D ? d : 0) * 2);
        q[i] = as_v8<M>(d < a.D ? x : u32x4{0, 0, 0, 0});
      }
    }
    const float to_log2 = (FP8 ? 1.0f : a.scale) * kLog2e;      // (8-bit keys: with the positions' scales)
    const float cap_in = a.softcap > 0.0f ? 2.0f * to_log2 / a.softcap : 0.0f, cap_out = a.softcap * kLog2e;
    constexpr float kLift = std::is_same_v<W, F16> ? 7.0f : 0.0f;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
    float m = kNegInf, l = 0.0f;
    bool bad = false;             // this lane has left values out that are no finite numbers

    const int32_t* const table = a.table + (int64_t)t.b * a.table_stride;
    const int last_entry = divided(max(hi - 1, 0), A.by_page);
    constexpr int kElem = FP8 ? 1 : 2;
    const char* const kbase = (const char*)a.k_cache + (int64_t)t.head * a.head_stride * kElem;
    const char* const vbase = (const char*)a.v_cache + (int64_t)t.head * a.head_stride * kElem;
    const int64_t page_bytes = a.page_stride * kElem, slot_bytes = a.slot_stride * kElem;
    const int slot = lane % F::kLanes, slot_row = lane / F::kLanes, row_bytes = a.D * kElem;
    auto lds_keys = [&](int buf) { return (Lds)&lds.tiles[wave][buf][0][0]; };
    auto lds_values = [&](int buf) { return (Lds)&lds.tiles[wave][buf][1][0]; };
    // What lies behind a key's last value is zeros, once for all.
    if (a.D < DP) {
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) {
        const int r = slot_row + i * F::kRows;
        if (F::key_piece(slot, r) * 16 >= row_bytes) {
#pragma unroll
          for (int b = 0; b < F::kBuffers; ++b) *(LdsPiece)(lds_keys(b) + r * F::kPitch + slot * 16) = u32x4{0, 0, 0, 0};
        }
      }
    }

    auto ask = [&](int sub) { return table[min(divided(walk.position(sub * kSub) + n, A.by_page), last_entry)]; };
    auto partial = [&](int pos0) {
      return pos0 + kSub - 1 > tile_lo || (a.window > 0 && pos0 <= low_of(tile_hi) && pos0 + kSub > a.keep_first);
    };
    u32x4 kreg[F::kLoads], vreg[F::kLoads];      // (those that do not go straight to LDS)
    float scale_of = 0.0f;        // of position n's key, in the upper half its value
    uint32_t loaded = 0;          // which positions of the loaded sub there are
    auto fetch = [&](int sub, int entry, int buf) {
      const int pos = walk.position(sub * kSub) + n, in_page = pos - divided(pos, A.by_page) * a.page_size;
      const int id = pos < hi && (uint32_t)entry < (uint32_t)a.num_pages ? entry : -1;
      loaded = (uint32_t)__ballot(id >= 0);
      if (half == 0) row_lds[wave][n] = max(id, 0) * page_bytes + (uint32_t)in_page * (uint64_t)(uint32_t)slot_bytes;
      if constexpr (FP8) {
        const int64_t s = a.scale_blocks == 0 ? t.head
                                              : ((int64_t)max(id, 0) * a.Hkv + t.head) * a.scale_blocks + divided(in_page, A.by_block);
        scale_of = id < 0 ? 0.0f : half == 0 ? a.k_scale[s] * a.scale : a.v_scale[s];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      int64_t at[F::kLoads];
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) at[i] = row_lds[wave][slot_row + i * F::kRows];
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) {
        const int piece = F::key_piece(slot, slot_row + i * F::kRows) * 16;
        if constexpr (!F::kDirect)
          kreg[i] = *(const u32x4*)(kbase + at[i] + (piece < row_bytes ? piece : 0));
        else if (piece < row_bytes)
          dma16(kbase + at[i] + piece, lds_keys(buf) + i * F::kRows * F::kPitch);
      }
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) {
        const int piece = F::value_piece(slot, slot_row + i * F::kRows) * 16;
        if constexpr (!F::kDirect)
          vreg[i] = *(const u32x4*)(vbase + at[i] + (piece < row_bytes ? piece : 0));
        else if (piece < row_bytes)
          dma16(vbase + at[i] + piece, lds_values(buf) + i * F::kRows * F::kPitch);
      }
    };

    const int quarter = (lane >> 4) & 1, l16 = lane & 15;
    // (8-bit values are read 8 x 16 at a time, 16-bit ones 4 x 16)
    const int value_row = FP8 ? half * 4 + (l16 >> 1) + (l16 >= 8 ? 4 : 0) : half * 4 + (l16 >> 2);
    const int value_at = value_row * F::kPitch + (FP8 ? l16 & 1 : l16 & 3) * 8, key_row = n * F::kPitch;
    int entry = 0;
    if (sub_begin + wave < sub_end) {
      fetch(sub_begin + wave, ask(sub_begin + wave), 0);
      entry = ask(sub_begin + wave + kWaves);
    }
    int buf = 0;
    for (int sub = sub_begin + wave; sub < sub_end; sub += kWaves) {
      const int pos0 = walk.position(sub * kSub);
      const uint32_t there = loaded;
      const bool look = partial(pos0);
      const Lds keys = lds_keys(buf), values = lds_values(buf);
      buf ^= F::kBuffers - 1;
      if constexpr (F::kDirect) {
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      } else {
#pragma unroll
        for (int i = 0; i < F::kLoads; ++i) {
          const int r = slot_row + i * F::kRows;
          if (F::key_piece(slot, r) * 16 < row_bytes) *(LdsPiece)(keys + r * F::kPitch + slot * 16) = kreg[i];
          *(LdsPiece)(values + r * F::kPitch + slot * 16) = vreg[i];
        }
      }
      if constexpr (FP8) scale_lds[wave][lane] = scale_of;
      if (sub + kWaves < sub_end) {
        fetch(sub + kWaves, entry, buf);
        entry = ask(sub + 2 * kWaves);
      }
      if (look || there != ~0u) {
        // Values as the product may have them.
#pragma unroll
        for (int i = 0; i < F::kLoads; ++i) {
          const int r = slot_row + i * F::kRows;
          const LdsPiece at = (LdsPiece)(values + r * F::kPitch + slot * 16);
          u32x4 v = *at;
          if (look && (FP8 ? drop_codes(v) : drop_others<W>(v)) && F::value_piece(slot, r) * 16 < row_bytes) bad = true;
          *at = (there >> r) & 1 ? v : u32x4{0, 0, 0, 0};
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      f32x16 x;
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        if constexpr (FP8) {
          const u32x2 c = *(LdsCodes)(keys + key_row + F::key_piece(i, n) * 16 + half * 8);
          x = M::mfma(fp8x8<M>(c[0], c[1]), q[i], x);
        } else {
          x = M::mfma(as_v8<M>(*(LdsPiece)(keys + key_row + F::key_piece(i * 2 + half, n) * 16)), q[i], x);
        }
      }

      if constexpr (FP8) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const f32x4 f = *(const f32x4*)&scale_lds[wave][j * 2 + half * 4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j + i] *= f[i];
        }
      }
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = capped(x[j] * cap_in, cap_out);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= to_log2;
      }
      uint32_t sees = ~0u;
      if (look || there != ~0u) {
        sees = bits_below(place + 1 - pos0) & (~bits_below(low + 1 - pos0) | bits_below(a.keep_first - pos0)) & there;
        sees >>= half * 4;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (!((sees >> (j / 4 * 8 + j % 4)) & 1)) x[j] = kNegInf;
      }
      float top = x[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) top = fmaxf(top, x[j]);
      top = over_halves_max(top);
      follow<std::is_same_v<W, F16>, false>(top, m, l, acc, m);
      const float ref = or_zero(m) - kLift;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // (two 16-bit terms of each weight, 16 bits of it: the matrix cores have the time)
        union { typename W::T e[8]; typename W::V8 v; } p, low;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          f32x4 f = {1.0f, 1.0f, 1.0f, 1.0f};
          if constexpr (FP8) f = *(const f32x4*)&scale_lds[wave][kSub + (j * 8 + i) * 2 + half * 4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = j * 8 + i + e;
            const float w = exp2_fast(x[at] - ref);
            l += w;
            // (a scale that is not seen may be anything)
            const float scaled = !FP8 ? w : ((sees >> (at / 4 * 8 + at % 4)) & 1) ? w * f[e] : 0.0f;
            p.e[i + e] = (typename W::T)scaled;
            low.e[i + e] = (typename W::T)(scaled - (float)p.e[i + e]);
          }
        }
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          typename W::V8 v;
          if constexpr (FP8) {
            const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(
                values + j * 16 * F::kPitch + value_at + F::value_piece(i * 2 + quarter, value_row) * 16));
            v = fp8x8<W>((uint32_t)c[0], (uint32_t)c[1]);
          } else {
            const Lds column = values + j * 16 * F::kPitch + value_at + F::value_pair(i * 2 + quarter, value_row) * 32;
            union { i16x4 h[2]; typename W::V8 v; } both;
            both.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)column);
            both.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(column + 8 * F::kPitch));
            v = both.v;
          }
          acc[i] = W::mfma(v, low.v, W::mfma(v, p.v, acc[i]));
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }

    // The four wavefronts' sums, relative to 2^ref each.
    l = over_halves_sum(l);
    const float ref = l == 0.0f ? kNegInf : or_zero(m) - kLift;
    if (half == 0) ml_lds[wave][n] = f32x2{ref, l};
    __syncthreads();
    auto joined = [&](int r) {
      float top = kNegInf, all = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml_lds[w][r][0]);
      const float at = or_zero(top);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all += ml_lds[w][r][1] * (ml_lds[w][r][1] == 0.0f ? 0.0f : exp2_fast(ml_lds[w][r][0] - at));
      return f32x2{all == 0.0f ? kNegInf : at, all};
    };
    const float f = l == 0.0f ? 0.0f : exp2_fast(ref - or_zero(joined(n)[0]));
    bad = __any(bad);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (wave == w) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f32x4* const to = (f32x4*)&sums[n][i * 32 + j * 8 + half * 4];
            f32x4 x = {acc[i][j * 4], acc[i][j * 4 + 1], acc[i][j * 4 + 2], acc[i][j * 4 + 3]};
            x *= f;
            *to = w == 0 ? x : *to + x;
          }
        }
        if (bad) {
          // What was left out, at the positions that a row sees (whatever its weight: an infinity stays one, or becomes NaN).
#pragma unroll 1
          for (int sub = sub_begin + wave; sub < sub_end; sub += kWaves) {
            const int pos0 = walk.position(sub * kSub);
            if (!partial(pos0)) continue;
#pragma unroll 1
            for (int pos = pos0; pos < min(pos0 + kSub, hi); ++pos) {
              const int in_table = divided(pos, A.by_page), id = table[in_table];
              if (!(pos <= place && (pos > low || pos < a.keep_first)) || (uint32_t)id >= (uint32_t)a.num_pages) continue;
              const char* const from = vbase + (int64_t)id * page_bytes + (int64_t)(pos - in_table * a.page_size) * slot_bytes;
#pragma unroll 1
              for (int d = half * 4; d < a.D; d += d % 4 == 3 ? 5 : 1) {
                union { uint16_t u; typename W::T t; } v;
                if constexpr (FP8)
                  v.t = fp8x8<W>(((const uint8_t*)from)[d], 0)[0];
                else
                  v.u = ((const uint16_t*)from)[d];
                if (!finite<W>(v.u)) sums[n][d] += (float)v.t;
              }
            }
          }
        }
      }
      __syncthreads();
    }
    const int quads = a.D / 4;
    const int64_t part = ((int64_t)t.slot * a.Hkv + t.head) * A.p.splits + t.split;
    for (int i = tid; i < kPromptFewRows * quads; i += 256) {
      const int r = i / quads, d = (i - r * quads) * 4, my_row = t.first + r;
      if (my_row >= t.rows) break;
      const f32x2 st = joined(r);
      const f32x4 x = *(const f32x4*)&sums[r][d];
      if (A.p.splits > 1) {
        if (d == 0) ((f32x2*)((char*)a.workspace + A.p.ml_at))[part * kPromptFewRows + r] = st;
        *(f32x4*)((float*)((char*)a.workspace + A.p.part_at) + (part * kPromptFewRows + r) * DP + d) = x;
      } else {
        const int my_tok = divided(my_row, A.by_group), hq = t.head * a.G + (my_row - my_tok * a.G);
        const int64_t out_row = (int64_t)(t.s0 + my_tok) * a.Hkv * a.G + hq;
        const float sink = a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf;
        const float top = or_zero(fmaxf(st[0], sink)), fix = st[1] == 0.0f ? 0.0f : exp2_fast(st[0] - top);
        const float total = st[1] * fix + exp2_fast(sink - top), inv = total == 0.0f ? 0.0f : fix / total;
        union { typename M::T e[4]; u32x2 u; } o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.e[e] = (typename M::T)(x[e] * inv);
        *(u32x2*)((char*)a.out + (out_row * a.D + d) * 2) = o.u;
        if (d == 0 && a.lse != nullptr) a.lse[out_row] = log_of_sum(top, total, a.sinks != nullptr ? a.sinks + hq : nullptr);
      }
    }
    // (the sums have been read when the next rows' keys come)
    if constexpr (AGAIN) __syncthreads();
    t.first += kPromptFewRows;
  } while (AGAIN && t.first < last_row);
}

// Joins the parts of tiles whose positions several workgroups shared: a lane holds 4 values of a row.  Where there are many
// parts, all of a workgroup's lanes have the same row and share them (`groups` of lanes); else each has a row.
template <class M>
__global__ __launch_bounds__(256) void prompt_attention_join_kernel(const KernelArgs A, int padded, int groups, int per_tile) {
  const PromptAttentionArgs& a = A.a;
  __shared__ f32x4 sum_lds[256];
  __shared__ f32x2 ml_lds[256 / 16];
  const int rest = blockIdx.x / per_tile, piece = blockIdx.x % per_tile;
  Tile t;
  KernelArgs one = A;
  one.p.splits = 1;
  one.by_splits = FastDiv{0, -1};
  if (!find_tile(one, rest, &t)) return;
  const int lanes = padded <= 64 ? 16 : padded <= 128 ? 32 : 64;      // of a row
  const int rows = 1 << A.p.row_shift, group = threadIdx.x / lanes, in_row = threadIdx.x % lanes, d = in_row * 4;
  const int at = groups > 1 ? piece : piece * (256 / lanes) + group, row = t.first + at;
  if (groups > 1 ? row >= t.rows : at >= rows || row >= t.rows || d >= a.D) return;      // (all lanes, where they meet below)
  const int tok = divided(row, A.by_group), hq = t.head * a.G + (row - tok * a.G);
  const int64_t slot = ((int64_t)t.slot * a.Hkv + t.head) * A.p.splits;
  const f32x2* const ml = (const f32x2*)((const char*)a.workspace + A.p.ml_at) + slot * rows + at;
  const float* const parts = (const float*)((const char*)a.workspace + A.p.part_at) + (slot * rows + at) * padded + (d < a.D ? d : 0);
  const int first = groups > 1 ? group : 0;
  float top = kNegInf;
#pragma unroll 4
  for (int s = first; s < A.p.splits; s += groups) top = fmaxf(top, ml[(int64_t)s * rows][0]);
  float total = 0.0f;
  f32x4 o = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = first; s < A.p.splits; s += groups) {
    const f32x2 x = ml[(int64_t)s * rows];
    if (x[1] == 0.0f) continue;          // (a part that saw nothing has left no sums)
    const float f = exp2_fast(x[0] - or_zero(top));
    total += x[1] * f;
    o += f * *(const f32x4*)(parts + (int64_t)s * rows * padded);
  }
  if (groups > 1) {
    sum_lds[threadIdx.x] = o;
    if (in_row == 0) ml_lds[group] = f32x2{top, total};
    __syncthreads();
    if (group > 0 || d >= a.D) return;
    float all = kNegInf;
    for (int i = 0; i < groups; ++i) all = fmaxf(all, ml_lds[i][0]);
    o = f32x4{0, 0, 0, 0};
    total = 0.0f;
    for (int i = 0; i < groups; ++i) {
      const f32x2 x = ml_lds[i];
      const float f = x[1] == 0.0f ? 0.0f : exp2_fast(x[0] - or_zero(all));
      total += x[1] * f;
      o += f * sum_lds[i * lanes + in_row];
    }
    top = all;
  }
  const float sink = a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf;
  const float ref = or_zero(fmaxf(top, sink)), fix = total == 0.0f ? 0.0f : exp2_fast(or_zero(top) - ref);
  total = total * fix + exp2_fast(sink - ref);
  const float inv = total == 0.0f ? 0.0f : fix / total;
  const int64_t out_row = (int64_t)(t.s0 + tok) * a.Hkv * a.G + hq;
  union { typename M::T e[4]; u32x2 u; } r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.e[e] = (typename M::T)(o[e] * inv);
  *(u32x2*)((char*)a.out + (out_row * a.D + d) * 2) = r.u;
  if (d == 0 && a.lse != nullptr) a.lse[out_row] = log_of_sum(ref, total, a.sinks != nullptr ? a.sinks + hq : nullptr);
}

int padded_width(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }

template <class M, bool FP8, int DP>
void launch_width(const KernelArgs& A, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)A.p.slots * A.a.Hkv * A.p.splits)), block(256);
  const int rows = 1 << A.p.row_shift;
  bool few = false;
  if constexpr (FP8 || DP <= kPromptFewWidth) {
    few = rows == kPromptFewRows;
    if (few) hipLaunchKernelGGL((prompt_attention_few_kernel<M, FP8, DP, false>), grid, block, 0, stream, A);
  }
  if (!few) hipLaunchKernelGGL((prompt_attention_kernel<M, FP8, DP>), grid, block, 0, stream, A);
  if (A.p.splits > 1) {
    const int lanes = DP <= 64 ? 16 : DP <= 128 ? 32 : 64;
    const int groups = A.p.splits >= 16 ? 256 / lanes : 1, per_tile = groups > 1 ? rows : rows / (256 / lanes);
    hipLaunchKernelGGL((prompt_attention_join_kernel<M>), dim3((unsigned)((int64_t)A.p.slots * A.a.Hkv * per_tile)), block, 0,
                       stream, A, DP, groups, per_tile);
  }
  if constexpr (FP8) {
    if (few) return;
    KernelArgs again = A;      // (a workgroup for every tile, with all of its positions)
    again.p.splits = 1;
    again.p.share = (A.a.max_len + kPromptKeys - 1) / kPromptKeys + 1;
    again.by_splits = fast_div(1);
    const dim3 tiles((unsigned)((int64_t)A.p.slots * A.a.Hkv));
    hipLaunchKernelGGL((prompt_attention_few_kernel<M, FP8, DP, true>), tiles, block, 0, stream, again);
  }
}

template <class M, bool FP8>
void launch_kind(const KernelArgs& A, hipStream_t stream) {
  switch (padded_width(A.a.D)) {
    case 64: launch_width<M, FP8, 64>(A, stream); break;
    case 96: launch_width<M, FP8, 96>(A, stream); break;
    case 128: launch_width<M, FP8, 128>(A, stream); break;
    case 192: launch_width<M, FP8, 192>(A, stream); break;
    default: launch_width<M, FP8, 256>(A, stream); break;
  }
}

}  // namespace

// Tiles of 32 rows where the sequences have no more on average; of wider 16-bit heads not (5 tokens of 32 sequences of up to
// 4096, 8 heads of 4 of 256: 481 us against 208, 127 registers spilled; of 192 values 186 against 178.  In 8 bits over up
// to 8192 267 against 485, and 223 against 436).
static int row_shift_of(int B, int tokens, int G, int D, bool fp8) {
  return (fp8 || D <= kPromptFewWidth) && (int64_t)tokens * G <= (int64_t)kPromptFewRows * B ? 5 : 7;
}

int64_t prompt_attention_slots(int B, int tokens, int G, int D, bool fp8) {
  return ((int64_t)tokens * G >> row_shift_of(B, tokens, G, D, fp8)) + B + 1;
}

PromptAttentionPlan prompt_attention_plan(int B, int tokens, int Hkv, int G, int D, int max_len, int window, int keep_first,
                                          bool fp8) {
  PromptAttentionPlan p{};
  p.row_shift = row_shift_of(B, tokens, G, D, fp8);
  p.slots = (int)prompt_attention_slots(B, tokens, G, D, fp8);
  const int rows = 1 << p.row_shift;
  // Where there are fewer tiles than the card holds workgroups, several share the positions of each.
  const int64_t tiles = (p.slots - 1) * (int64_t)Hkv;
  int64_t seen = max_len;
  if (window > 0) seen = std::min<int64_t>(max_len, (int64_t)window + rows + 16 + std::min(keep_first, max_len) + kPromptKeys);
  // Shares of one size for all sequences (those behind a shorter one's end are empty; shares by a sequence's own length
  // are no faster).  How many: 5 tokens over 1024 to 8192 positions of 32 sequences in 8 bits, 8 heads of 4, take 114 us
  // with 1024 workgroups, 111 with 2048, 101 with 4096, 113 with 8192; 64 over the same, in tiles of 128 rows, 105 with
  // 1024, 110 with 2048, 146 with 512.  At most 64, which one launch joins.
  const int64_t keys = std::max<int64_t>(1, (seen + kPromptKeys - 1) / kPromptKeys);
  const int64_t wanted = rows == kPromptFewRows ? 4096 : 1024;
  const int64_t splits = std::max<int64_t>(1, std::min({keys / 4, wanted / tiles, (int64_t)64}));
  p.share = (int)((keys + splits - 1) / splits);
  if (rows == kPromptFewRows) p.share = (p.share + 1) / 2 * 2;      // (two for each wavefront of two subs)
  p.splits = (int)((keys + p.share - 1) / p.share);
  size_t at = 0;
  auto part = [&at](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
  if (p.splits > 1) {
    const size_t all = (size_t)p.slots * Hkv * p.splits * rows;
    p.ml_at = part(all * 8);
    p.part_at = part(all * padded_width(D) * 4);
  }
  p.bytes = at;
  return p;
}

void launch_prompt_attention(const PromptAttentionArgs& a, int kind, hipStream_t stream) {
  KernelArgs A{};
  A.a = a;
  A.p = prompt_attention_plan(a.B, a.tokens, a.Hkv, a.G, a.D, a.max_len, a.window, a.keep_first, kind >= kKvFp8Bf16);
  A.by_page = fast_div(a.page_size);
  A.by_block = fast_div(a.scale_blocks > 0 ? a.page_size / a.scale_blocks : 1);
  A.by_group = fast_div(a.G);
  A.by_heads = fast_div(a.Hkv);
  A.by_splits = fast_div(A.p.splits);
  switch (kind) {
    case kKvBf16: launch_kind<Bf16, false>(A, stream); break;
    case kKvF16: launch_kind<F16, false>(A, stream); break;
    case kKvFp8Bf16: launch_kind<Bf16, true>(A, stream); break;
    default: launch_kind<F16, true>(A, stream); break;
  }
}

}  // namespace vk

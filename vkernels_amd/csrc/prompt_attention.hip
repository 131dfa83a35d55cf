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

constexpr int kWaves = 4, kWaveRows = kPromptRows / kWaves;
static_assert(kWaveRows == 32, "a wavefront's rows are the columns of a matrix instruction");

struct KernelArgs {
  PromptAttentionArgs a;
  PromptAttentionPlan p;
  FastDiv by_page, by_block, by_group, by_heads, by_splits;
};

// What a workgroup works on.
struct Tile {
  int b;             // the sequence; B: rows behind the last one
  int slot, head, split;
  int s0, tokens;    // the sequence's first row of q, and how many it has
  int first, rows;   // its first row of the tile, and rows of the sequence
};
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
  // The tiles of sequence b begin at start rows / 128 + b: it has at most as many as lie up to the next one's.
  auto base = [&](int i) { return start(i) * a.G / kPromptRows + i; };
  t->b = __builtin_amdgcn_readfirstlane(last_not_above(a.B + 1, t->slot, base));
  const int k = t->slot - base(t->b);
  t->s0 = start(t->b);
  t->tokens = (t->b < a.B ? max(start(t->b + 1), t->s0) : a.tokens) - t->s0;
  t->first = k * kPromptRows;
  t->rows = t->tokens * a.G;
  return k >= 0 && t->first < t->rows;
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

template <bool FP8, int DP>
struct Layout {
  static constexpr int kPieces = DP / 8;                       // of a row: 8 values
  static constexpr int kLanes = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;   // threads that load a row
  static constexpr int kPass = 256 / kLanes;                   // rows that the workgroup loads at once
  static constexpr int kLoads = kPromptKeys / kPass;
  // Keys: 16 bytes behind each row, so that 16 rows' pieces lie in different banks.  Values: rows of a power of two
  // pieces, pairs of them exchanged by the row for the transposed reads.
  static constexpr int kKeyPitch = DP * 2 + 16, kValuePitch = kLanes * 16;
  static constexpr int kKeyBytes = kPromptKeys * kKeyPitch, kValueBytes = kPromptKeys * kValuePitch;
  static constexpr int kBuffer = kKeyBytes + kValueBytes;
  static constexpr int kLds = 2 * kBuffer;
  static __device__ __forceinline__ int turn(int row) { return DP <= 64 ? (row >> 1) & 3 : row & 7; }
};

// Is a 16-bit value (in the lower half of x) a finite number?
template <class W>
__device__ __forceinline__ bool finite(uint32_t x) {
  constexpr uint32_t kExponent = std::is_same_v<W, F16> ? 0x7C00u : 0x7F80u;
  return (x & kExponent) != kExponent;
}

// S^T = K q^T and O^T += V^T P^T, both 32 x 32 x 16 with the keys (the head's width) as rows and a wavefront's 32
// rows as columns: a lane holds half of one row's scores, so that maximum, sum and rescaling stay in the lane and its
// neighbour 32 lanes on, and its weights are where the second product wants them, in the order of positions in
// which the values are read from LDS (transposed, 4 x 16 at a time).
// Keys and values of 64 positions go to LDS through registers, a tile ahead, in two buffers.
template <class M, bool FP8, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void prompt_attention_kernel(const KernelArgs A) {
  typedef Layout<FP8, DP> L;
  typedef std::conditional_t<FP8, Bf16, M> W;      // what weights and values are multiplied in
  typedef std::conditional_t<FP8, u32x2, u32x4> Piece;
  const PromptAttentionArgs& a = A.a;
  __shared__ __attribute__((aligned(16))) char lds[L::kLds];
  __shared__ __attribute__((aligned(16))) float scale_lds[FP8 ? 2 : 1][kWaves][2][kPromptKeys];
  __shared__ int64_t row_lds[kWaves][kPromptKeys];
  __shared__ uint32_t any_bad;      // values that are no finite numbers have been left out

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile t;
  if (!find_tile(A, blockIdx.x, &t)) return;
  const int Hq = a.Hkv * a.G;
  if (t.b == a.B) {
    // Rows that belong to no sequence.
    if (!a.clear_rest || t.split > 0) return;
    const int pieces = a.D / 8;
    for (int i = tid; i < kPromptRows * pieces; i += 256) {
      const int r = t.first + i / pieces, tok = divided(r, A.by_group);
      if (r >= t.rows) break;
      const int64_t row = (int64_t)(t.s0 + tok) * Hq + t.head * a.G + (r - tok * a.G);
      *(u32x4*)((char*)a.out + (row * a.D + i % pieces * 8) * 2) = u32x4{0, 0, 0, 0};
      if (i % pieces == 0 && a.lse != nullptr) a.lse[row] = kNegInf;
    }
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
  const int share = (walk.tiles + A.p.splits - 1) / A.p.splits;
  const int tile_begin = t.split * share, tile_end = min(walk.tiles, tile_begin + share);

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
  const bool plain = !FP8 && !(a.softcap > 0.0f) && a.scale > 0.0f;
  const float to_log2 = k_scale * kLog2e;
  const float cap_in = a.softcap > 0.0f ? 2.0f * k_scale * kLog2e / a.softcap : 0.0f, cap_out = a.softcap * kLog2e;

  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
  float m = kNegInf, l = 0.0f;
  // (fp16 weights end at 2^-24: they are kept 2^7 above the reference, so that with the slack they reach 2^15)
  constexpr float kLift = std::is_same_v<W, F16> ? 7.0f : 0.0f;

  // What lies behind a row's last value is zeros, once for all.
  if (a.D < DP) {
    const int empty = L::kPieces - a.D / 8;
    for (int i = tid; i < 2 * kPromptKeys * empty; i += 256) {
      const int buf = i / (kPromptKeys * empty), r = i / empty % kPromptKeys;
      *(u32x4*)(lds + buf * L::kBuffer + r * L::kKeyPitch + (a.D / 8 + i % empty) * 16) = u32x4{0, 0, 0, 0};
    }
  }

  const int32_t* const table = a.table + (int64_t)t.b * a.table_stride;
  const int last_entry = divided(max(hi - 1, 0), A.by_page);
  constexpr int kElem = FP8 ? 1 : 2;
  const char* const kbase = (const char*)a.k_cache + (int64_t)t.head * a.head_stride * kElem;
  const char* const vbase = (const char*)a.v_cache + (int64_t)t.head * a.head_stride * kElem;
  const int64_t page_bytes = a.page_stride * kElem, slot_bytes = a.slot_stride * kElem;
  const int piece = tid % L::kLanes, piece_row = tid / L::kLanes;
  const bool has_piece = piece * 8 < a.D;
  const int piece_at = has_piece ? piece * 8 * kElem : 0;

  // The page of position lane of a tile, asked for a tile ahead; -1 where there is none.
  auto ask = [&](int tile) {
    const int pos = walk.position(tile * kPromptKeys) + lane;
    const int id = table[min(divided(pos, A.by_page), last_entry)];
    return pos < hi && (uint32_t)id < (uint32_t)a.num_pages ? id : -1;
  };
  Piece kreg[L::kLoads], vreg[L::kLoads];
  float ks = 1.0f, vs = 1.0f;
  uint64_t loaded = 0;         // which positions of the loaded tile there are
  auto fetch = [&](int tile, int ids) {
    // A lane works out where its position's rows lie, for the wavefront's lanes that load them.
    const int pos = walk.position(tile * kPromptKeys) + lane, slot = pos - divided(pos, A.by_page) * a.page_size;
    loaded = __ballot(ids >= 0);
    row_lds[wave][lane] = max(ids, 0) * page_bytes + (uint32_t)slot * (uint64_t)(uint32_t)slot_bytes;
    if constexpr (FP8) {
      const int64_t at = a.scale_blocks == 0 ? t.head
                                             : ((int64_t)max(ids, 0) * a.Hkv + t.head) * a.scale_blocks + divided(slot, A.by_block);
      ks = ids >= 0 ? a.k_scale[at] * a.scale : 0.0f;
      vs = ids >= 0 ? a.v_scale[at] : 0.0f;
    }
    // (lanes read what other lanes of their wavefront wrote: LDS keeps the order, and so must the compiler)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    int64_t at[L::kLoads];
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) at[i] = row_lds[wave][piece_row + i * L::kPass] + piece_at;
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      kreg[i] = *(const Piece*)(kbase + at[i]);
      vreg[i] = *(const Piece*)(vbase + at[i]);
    }
  };
  // Does any row of the workgroup not see all of a tile?
  auto partial = [&](int pos0) {
    return pos0 + kPromptKeys - 1 > tile_lo ||
           (a.window > 0 && pos0 <= low_of(tile_hi) && pos0 + kPromptKeys > a.keep_first);
  };
  // The loaded tile to LDS: positions that there are not as zeros.  Where some rows do not see all of it, so are values
  // that are no finite numbers: a weight of 0 times them would not be 0 (they are added in the end).
  auto put = [&](int buf, int tile) {
    char* const to = lds + buf * L::kBuffer;
    const bool look = partial(walk.position(tile * kPromptKeys));
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      const int r = piece_row + i * L::kPass;
      u32x4 k, v;
      if constexpr (FP8) {
        union { typename M::V8 v; u32x4 u; } kc;
        union { typename W::V8 v; u32x4 u; } vc;
        kc.v = fp8x8<M>(kreg[i][0], kreg[i][1]);
        vc.v = fp8x8<W>(vreg[i][0], vreg[i][1]);
        k = kc.u;
        v = vc.u;
      } else {
        k = kreg[i];
        v = vreg[i];
      }
      if (!((loaded >> r) & 1)) v = u32x4{0, 0, 0, 0};
      if (look) {
        // (an exponent of ones carries into the half's sign)
        constexpr uint32_t kExponents = std::is_same_v<W, F16> ? 0x7C007C00u : 0x7F807F80u;
        constexpr uint32_t kOnes = std::is_same_v<W, F16> ? 0x04000400u : 0x00800080u;
        uint32_t all = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = ((v[e] & kExponents) + kOnes) & 0x80008000u;
          v[e] &= ~((bad >> 15) * 0xFFFFu);
          all |= bad;
        }
        if (all != 0 && has_piece) any_bad = 1;
      }
      if (has_piece) {
        *(u32x4*)(to + r * L::kKeyPitch + piece * 16) = k;
        *(u32x4*)(to + L::kKeyBytes + r * L::kValuePitch + ((piece >> 1) ^ L::turn(r)) * 32 + (piece & 1) * 16) = v;
      }
    }
    if constexpr (FP8) {
      scale_lds[buf][wave][0][lane] = ks;
      scale_lds[buf][wave][1][lane] = vs;
    }
  };

  const int quarter = (lane >> 4) & 1, l16 = lane & 15;
  const int value_row = half * 4 + (l16 >> 2), value_turn = L::turn(value_row);
  uint64_t there = 0;
  if (tid == 0) any_bad = 0;
  if (tile_begin < tile_end) {
    fetch(tile_begin, ask(tile_begin));
    int ids = ask(tile_begin + 1);
    __syncthreads();
    put(0, tile_begin);
    there = loaded;
    if (tile_begin + 1 < tile_end) {
      fetch(tile_begin + 1, ids);
      ids = ask(tile_begin + 2);
    }
    __syncthreads();
    for (int tile = tile_begin; tile < tile_end; ++tile) {
      const int buf = (tile - tile_begin) & 1;
      const char* const keys = lds + buf * L::kBuffer;
      const int pos0 = walk.position(tile * kPromptKeys);
      // Hidden from every row of the wavefront: behind the last one's place, or in front of the first one's window.
      const bool skip = pos0 > wave_hi || (pos0 + kPromptKeys - 1 <= wave_low && pos0 >= a.keep_first) || wave_first >= t.rows;
      float x[32];
      if (!skip) {
        f32x16 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
          for (int j = 0; j < 16; ++j) s[kt][j] = 0.0f;
          const char* const from = keys + (kt * 32 + n) * L::kKeyPitch + half * 16;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) s[kt] = M::mfma(as_v8<M>(*(const u32x4*)(from + i * 32)), q[i], s[kt]);
#pragma unroll
          for (int j = 0; j < 16; ++j) x[kt * 16 + j] = s[kt][j];
        }
      }
      const bool more = tile + 1 < tile_end;
      const uint64_t these = there;
      if (more) {
        put(buf ^ 1, tile + 1);
        there = loaded;
        if (tile + 2 < tile_end) {
          fetch(tile + 2, ids);
          ids = ask(tile + 3);
        }
      }
      if (!skip) {
        // Scores in powers of two, unless they are taken there with the reference.
        float c = to_log2;
        if (!plain) {
          c = 1.0f;
          if constexpr (FP8) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const f32x4 f = *(const f32x4*)&scale_lds[buf][wave][0][j / 16 * 32 + j % 16 / 4 * 8 + half * 4];
#pragma unroll
              for (int i = 0; i < 4; ++i) x[j + i] *= f[i];
            }
          }
          if (a.softcap > 0.0f) {
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = capped(x[j] * cap_in, cap_out);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] *= to_log2;
          }
        }
        const bool whole = these == ~0ull && pos0 + kPromptKeys - 1 <= wave_lo &&
                           (a.window <= 0 || pos0 > low_of(wave_hi) || pos0 + kPromptKeys <= a.keep_first);
        uint64_t sees = ~0ull;      // the positions of the tile that this lane's row sees
        if (!whole) {
          auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
          sees = below(place + 1 - pos0) & (~below(low + 1 - pos0) | below(a.keep_first - pos0)) & these;
          const uint64_t mine = sees >> (half * 4);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int r = j / 16 * 32 + j % 16 / 4 * 8 + j % 4;
            if (!((mine >> r) & 1)) x[j] = kNegInf;
          }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 32; ++j) top = fmaxf(top, x[j]);
        const u32x2 both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * c;
        if (__any(top > m + kSlack)) {
          // (a row by itself: what it gives does not depend on the rows beside it)
          const float m_new = top > m + kSlack ? top : m;
          const float fix = exp2_fast(m - or_zero(m_new));
          m = m_new;
          l *= fix;
#pragma unroll
          for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[i][j] *= fix;
        }
        const float ref = or_zero(m) - kLift;
        // Weights of 16 bits (half a step of their type is what the result is off by from each, as from its own
        // rounding); their sum is of those in 32.
        union { typename W::T e[32]; typename W::V8 v[4]; } p;
        auto weigh = [&](auto all) {
          const uint64_t mine = sees >> (half * 4);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            f32x4 f = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (FP8) f = *(const f32x4*)&scale_lds[buf][wave][1][j / 16 * 32 + j % 16 / 4 * 8 + half * 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = exp2_fast(__builtin_fmaf(x[j + i], c, -ref));
              l += w;
              // (a scale that is not seen may be anything)
              const float scaled = FP8 ? decltype(all)::value || ((mine >> (j / 16 * 32 + j % 16 / 4 * 8 + i)) & 1) ? w * f[i] : 0.0f : w;
              p.e[j + i] = (typename W::T)scaled;
            }
          }
        };
        if (!FP8 || whole) weigh(std::true_type{}); else weigh(std::false_type{});
        const char* const values = keys + L::kKeyBytes + value_row * L::kValuePitch + (l16 & 3) * 8;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const char* const column = values + ((i * 2 + quarter) ^ value_turn) * 32;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            union { i16x4 h[2]; typename W::V8 v; } v;
            v.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4*)(column + j * 16 * L::kValuePitch));
            v.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4*)(column + (j * 16 + 8) * L::kValuePitch));
            acc[i] = W::mfma(v.v, p.v[j], acc[i]);
          }
        }
      }
      __syncthreads();
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

  // The sums of a row: this lane's positions and those of the lane 32 on.
  {
    const u32x2 both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  }
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

// Joins the parts of tiles whose positions several workgroups shared: a lane holds 4 values of a row.
template <class M>
__global__ __launch_bounds__(256) void prompt_attention_join_kernel(const KernelArgs A, int padded, int per_tile) {
  const PromptAttentionArgs& a = A.a;
  const int rest = blockIdx.x / per_tile, part = blockIdx.x % per_tile;
  Tile t;
  KernelArgs one = A;
  one.p.splits = 1;
  one.by_splits = FastDiv{0, -1};
  if (!find_tile(one, rest, &t) || t.b == a.B) return;
  const int lanes = padded <= 64 ? 16 : padded <= 128 ? 32 : 64;      // of a row
  const int at = part * (256 / lanes) + threadIdx.x / lanes, d = threadIdx.x % lanes * 4, row = t.first + at;
  if (at >= kPromptRows || row >= t.rows || d >= a.D) return;
  const int tok = divided(row, A.by_group), hq = t.head * a.G + (row - tok * a.G);
  const int64_t slot = ((int64_t)t.slot * a.Hkv + t.head) * A.p.splits;
  const f32x2* const ml = (const f32x2*)((const char*)a.workspace + A.p.ml_at) + slot * kPromptRows + at;
  const float* const parts = (const float*)((const char*)a.workspace + A.p.part_at) + (slot * kPromptRows + at) * padded + d;
  const float sink = a.sinks != nullptr ? a.sinks[hq] * kLog2e : kNegInf;
  float top = sink;
  for (int s = 0; s < A.p.splits; ++s) top = fmaxf(top, ml[s * kPromptRows][0]);
  top = or_zero(top);
  float total = exp2_fast(sink - top);
  f32x4 o = {0, 0, 0, 0};
  for (int s = 0; s < A.p.splits; ++s) {
    const f32x2 x = ml[s * kPromptRows];
    if (x[1] == 0.0f) continue;          // (a part that saw nothing has left no sums)
    const float f = exp2_fast(x[0] - top);
    total += x[1] * f;
    o += f * *(const f32x4*)(parts + (int64_t)s * kPromptRows * padded);
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t out_row = (int64_t)(t.s0 + tok) * a.Hkv * a.G + hq;
  union { typename M::T e[4]; u32x2 u; } r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.e[e] = (typename M::T)(o[e] * inv);
  *(u32x2*)((char*)a.out + (out_row * a.D + d) * 2) = r.u;
  if (d == 0 && a.lse != nullptr) a.lse[out_row] = log_of_sum(top, total, a.sinks != nullptr ? a.sinks + hq : nullptr);
}

int padded_width(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }

template <class M, bool FP8, int DP>
void launch_width(const KernelArgs& A, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)A.p.slots * A.a.Hkv * A.p.splits)), block(256);
  hipLaunchKernelGGL((prompt_attention_kernel<M, FP8, DP>), grid, block, 0, stream, A);
  if (A.p.splits > 1) {
    const int per_tile = kPromptRows / (256 / (DP <= 64 ? 16 : DP <= 128 ? 32 : 64));
    hipLaunchKernelGGL((prompt_attention_join_kernel<M>), dim3((unsigned)((int64_t)A.p.slots * A.a.Hkv * per_tile)), block, 0,
                       stream, A, DP, per_tile);
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

int64_t prompt_attention_slots(int B, int tokens, int G) { return (int64_t)tokens * G / kPromptRows + B + 1; }

PromptAttentionPlan prompt_attention_plan(int B, int tokens, int Hkv, int G, int D, int max_len, int window, int keep_first) {
  PromptAttentionPlan p{};
  p.slots = (int)prompt_attention_slots(B, tokens, G);
  // Where there are fewer tiles than the card holds workgroups, several share the positions of each.
  const int64_t tiles = ((int64_t)tokens * G / kPromptRows + std::min(B, tokens)) * Hkv;
  int64_t seen = max_len;
  if (window > 0) seen = std::min<int64_t>(max_len, (int64_t)window + kPromptRows + 16 + std::min(keep_first, max_len) + kPromptKeys);
  const int64_t most = std::max<int64_t>(1, seen / (4 * kPromptKeys));
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, 1024 / std::max<int64_t>(1, tiles)));
  size_t at = 0;
  auto part = [&at](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
  if (p.splits > 1) {
    const size_t rows = (size_t)p.slots * Hkv * p.splits * kPromptRows;
    p.ml_at = part(rows * 8);
    p.part_at = part(rows * padded_width(D) * 4);
  }
  p.bytes = at;
  return p;
}

void launch_prompt_attention(const PromptAttentionArgs& a, int kind, hipStream_t stream) {
  KernelArgs A{};
  A.a = a;
  A.p = prompt_attention_plan(a.B, a.tokens, a.Hkv, a.G, a.D, a.max_len, a.window, a.keep_first);
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

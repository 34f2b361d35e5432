// Units of attention over the 8-bit cache (kv_cache.h) and how their work is shared out: what the kernels
// of cache_attn.hip have in common with those that join their partial results (prefix_attn.hip).
#pragma once

#include "attn_tiles.h"
#include "kv_cache.h"

#include <math.h>

namespace vdn {
namespace units {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kTile = 64;              // tokens of a wave's step
constexpr int kQuad = kTile * kWaves;  // tokens of a workgroup's step

// Units of tables of up to so many quads are not split: the second step costs less than the join.
// 128 sequences of 100 - 300 tokens, 32 heads on 8: 22.5 us against 25.6; one of 500, 56 heads: 8.7,
// 10.3. With four quads 64 of 100 - 1000 tokens take 26.9 against 25.0, one of 1000 12.4 against 10.5.
constexpr int kWholeQuads = 2;

// Workgroups that share a CU, by the registers that a tile's codes, Q and O take: one for wide heads
// or 32 rows, three for 64 channels (128 sequences of 100 - 300 tokens, 8 K/V heads: 17.4 us
// against 20.5 with two; long sequences the same).
constexpr int workgroups_per_cu(int head_dim, int rows) {
  return head_dim * rows > 128 * 16 ? 1 : head_dim * rows > 64 * 16 ? 2 : 3;
}

struct Queries {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;  // sequence / token / head strides (elements)
  int tokens, group;                           // Q, G
};

struct Lengths {
  const int* table;
  const int* lengths;
  int64_t t_st, t_sh;   // sequence / K/V head strides of the table (0: one row for all heads)
  int batch, width;
};

// Workspace slots: two per workgroup (its first and its last unfinished unit), each kRows rows
// of D + 4 floats (O, m, l, two unused).
struct Split {
  float* slots;   // null: units are not split
  int workgroups;
  int unit_cost;
};

__device__ __forceinline__ int seq_tokens(const KvCache& c, const Lengths& s, int b) {
  const int64_t most = static_cast<int64_t>(s.width) << c.log_page;
  return static_cast<int>(min(static_cast<int64_t>(max(s.lengths[b], 0)), most));
}

__device__ __forceinline__ int quads_of(int tokens) { return max((tokens + kQuad - 1) / kQuad, 1); }

// What a unit counts for when the work is shared out: its quads, and in front of them unit_cost for its
// queries, its first loads' latency and the join of the waves. One quad where units are split: 64
// sequences of 100 - 1000 tokens, 32 heads on 8: 22.4 us against 25.0 with quads alone, 16 of 100 - 4097
// with 12 heads x 64 18.1, 19.9; even ones the same (two: 64 of 100 - 2048 tokens 30.7, 28.6). Nothing
// where they stay whole: 128 of 100 - 300 tokens 22.0, 23.2.
constexpr int kUnitCost = 1;
__device__ __forceinline__ int cost_of(const Split& sp, int tokens) { return quads_of(tokens) + sp.unit_cost; }

// Workgroup w of n has the positions share_from(w) .. share_from(w + 1) - 1 of `total` >= n, x is one of
// share_of(x)'s. Rounded up: where a whole number of workgroups share a unit, they have as many quads each.
__device__ __forceinline__ int64_t share_from(int64_t total, int n, int w) { return (total * w + n - 1) / n; }
__device__ __forceinline__ int64_t share_of(int64_t total, int n, int64_t x) { return x * n / total; }

// Where a workgroup's share of all units' costs begins (sequence b: units times its cost), from a
// prefix over the lengths. Every wave does it for itself, 64 strips of sequences at a time: no
// barrier, and for up to 64 sequences one load.
struct Place {
  int64_t from, to;   // the workgroup's share (none: from = to)
  int64_t before;   // costs in front of sequence seq
  int seq;
};

__device__ __forceinline__ int wave_prefix(int x, int lane) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int other = __shfl_up(x, d);
    x += lane >= d ? other : 0;
  }
  return x;
}

__device__ inline Place find_share(const KvCache& c, const Lengths& s, const Split& sp, int units, int wg) {
  const int lane = threadIdx.x & 63;
  const int strip = (s.batch + 63) / 64;
  const int b0 = min(lane * strip, s.batch), b1 = min(b0 + strip, s.batch);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += cost_of(sp, seq_tokens(c, s, b));
  const int incl = wave_prefix(mine, lane);
  Place p;
  const int64_t total = static_cast<int64_t>(__builtin_amdgcn_readlane(incl, 63)) * units;
  const int n_wg = static_cast<int>(min(total, static_cast<int64_t>(sp.workgroups)));
  p.from = wg < n_wg ? share_from(total, n_wg, wg) : total;
  p.to = wg < n_wg ? share_from(total, n_wg, wg + 1) : total;
  const int64_t at = p.from;
  // the strip, then the sequence inside it
  const int front = __popcll(__ballot(static_cast<int64_t>(incl) * units <= at));
  const int owner = min(front, 63);
  int before = __builtin_amdgcn_readlane(incl - mine, owner);
  int seq = __builtin_amdgcn_readlane(b0, owner);
  if (strip > 1) {
    const int last = min(seq + strip, s.batch) - 1;
    for (; seq < last; ++seq) {
      const int n = cost_of(sp, seq_tokens(c, s, seq));
      if (at < static_cast<int64_t>(before + n) * units) break;
      before += n;
    }
  }
  p.before = static_cast<int64_t>(before) * units;
  p.seq = seq;
  return p;
}

template <bool kF16>
struct Half;

template <>
struct Half<false> {
  typedef bf16x8 x8;
  template <bool kHi>
  static __device__ __forceinline__ uint32_t widen2(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, kHi));
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ uint32_t pack_out(float a, float b) { return pack(a, b); }
};

template <>
struct Half<true> {
  typedef f16x8 x8;
  template <bool kHi>
  static __device__ __forceinline__ uint32_t widen2(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, kHi));
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return f32_to_f16_bits(a) | static_cast<uint32_t>(f32_to_f16_bits(b)) << 16;
  }
  // An output: E4M3 takes values next to fp16's largest one to 65536, which would be an infinity.
  static __device__ __forceinline__ uint32_t pack_out(float a, float b) {
    return pack(f16_in_range(a), f16_in_range(b));
  }
};

// Eight codes -> eight 16-bit values of code * s (s a power of two).
template <bool kF16>
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float s) {
  return u32x4{Half<kF16>::template widen2<false>(lo, s), Half<kF16>::template widen2<true>(lo, s),
               Half<kF16>::template widen2<false>(hi, s), Half<kF16>::template widen2<true>(hi, s)};
}

// The first `n` (0 .. 4) bytes of a word.
__device__ __forceinline__ uint32_t first_bytes(int n) {
  return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
}

// Bytes of w that hold the NaN code, as 0x38 (1.0) in the same place and 0 elsewhere.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (((w >> (8 * i)) & 0x7fu) == 0x7fu) out |= 0x38u << (8 * i);
  return out;
}

// Factor of a row's output from its sum of weights and the number of keys that it sees. No weights: a row
// that sees no key is zero, one whose scores are all -inf has no softmax and is NaN.
__device__ __forceinline__ float inverse_of(float sum, int keys) {
  return sum == 0.f ? (keys > 0 ? NAN : 0.f) : 1.0f / sum;
}

// ---- host ----

// How vdn_cache_attention cuts its work: rows of a row block, and whether units are split.
struct UnitPlan {
  int block, row_blocks;
  bool split;
  Split sp;             // slots to be set by the caller
  int64_t slot_bytes;   // of a split's slots
};
UnitPlan plan_units(int batch, int width, int log_page, int64_t rows, int kv_heads, int head_dim);

// The same with every unit's maximum, sum and O left in fp32 instead of an output: a split unit's in the
// slots, a whole one's rows in whole[(b tokens + i) heads + h][D + 4]. The sizes have to be checked.
int launch_partials(const KvCache& c, const Queries& io, const Lengths& s, const UnitPlan& plan, float* whole,
                    int head_dim, int dtype, float scale_log2, hipStream_t stream);

}  // namespace units
}  // namespace vdn

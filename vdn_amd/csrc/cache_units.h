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
  // Beside other work of the same launch (prefix_attn.hip): the workgroups that the card has left beside it
  // (0: none, or no such work), and how long each of its own takes, in quads.
  int few;
  float beside;
};

// Whether `total` costs are better shared by the few workgroups beside the other work, because they end sooner
// than both one after the other. (A quad takes less time where not all ask for codes.)
__host__ __device__ __forceinline__ bool few_suffice(const Split& sp, int64_t total) {
  const float cost = static_cast<float>(total), few = 0.7f * cost / sp.few;
  return sp.few > 0 && (few > sp.beside ? few : sp.beside) < sp.beside + cost / sp.workgroups;
}

// How many workgroups share `total` costs: all (kBeside: behind the other work, or the few).
template <bool kBeside>
__device__ __forceinline__ int sharers(const Split& sp, int64_t total) {
  const int n = kBeside && few_suffice(sp, total) ? min(sp.workgroups, sp.few) : sp.workgroups;
  return static_cast<int>(min(total, static_cast<int64_t>(n)));
}

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

template <bool kBeside>
__device__ inline Place find_share(const KvCache& c, const Lengths& s, const Split& sp, int units, int wg) {
  const int lane = threadIdx.x & 63;
  const int strip = (s.batch + 63) / 64;
  const int b0 = min(lane * strip, s.batch), b1 = min(b0 + strip, s.batch);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += cost_of(sp, seq_tokens(c, s, b));
  const int incl = wave_prefix(mine, lane);
  Place p;
  const int64_t total = static_cast<int64_t>(__builtin_amdgcn_readlane(incl, 63)) * units;
  const int n_wg = sharers<kBeside>(sp, total);
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

// Unit wg, whole, as a share of its own.
__device__ __forceinline__ Place place_of(const KvCache& c, const Lengths& s, const Split& sp, int units, int wg) {
  const int b = wg / units;
  const int64_t at = static_cast<int64_t>(wg - b * units) * cost_of(sp, seq_tokens(c, s, b));
  return Place{at, at + 1, 0, b};
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
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
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

// What a workgroup does: its share of all units (workgroup wg of sp.workgroups), with one table a sequence or one
// a K/V head; unit wg, whole, with one a K/V head; or its share beside other work, with nothing
// divided by the sums: a whole unit's rows go to `part` as a slot's do ([row][D + 4]); or the same with a unit for
// each wave, whole (short tables: the waves have nothing to join, and four units are under way at a time).
enum Mode { kShare, kShareHeads, kOneEach, kParts, kPartsByWave };

// Few query rows of a prefix (prefix_attn.hip), which a workgroup takes like a unit, its waves the tiles
// in turn: rows row .. + rows of the sequences behind it, tiles from .. to of `tokens`, which all rows see.
struct FewRows {
  const int* table;
  float* slot;
  int first, row, rows, head, from, to, tokens;
};

// In front of a launch's workgroups there may be others with work of their own (kParts): Front::workgroups of them,
// Front::run is what they do, and kPerCu of either fit a CU. (The body stands in the kernel itself: as a function
// that two kernels call it took a hundred more scalar spills and 2 - 5% more time.)
struct NoFront {
  static constexpr int kPerCu = 0;
};

template <int kD, int kNR, bool kF16, Mode kMode, class Front>
__global__ void __launch_bounds__(kThreads, Front::kPerCu > 0 ? Front::kPerCu : workgroups_per_cu(kD, 16 * kNR))
cache_attn_kernel(KvCache c, Queries io, Lengths s, Split sp, int row_blocks, float scale_log2, float* part,
                  Front front) {
  constexpr bool kByWave = kMode == kPartsByWave, kPart = kMode == kParts || kByWave;
  int wg = blockIdx.x;
  [[maybe_unused]] FewRows few{};
  bool is_few = false;
  if constexpr (kPart) {
    if (wg < front.workgroups) {
      is_few = front.run(c, io, scale_log2, wg, few);
      if (!is_few) return;
    }
    wg -= front.workgroups;
  }
  constexpr int kRows = 16 * kNR;     // query rows of a unit
  constexpr int kKL = kD / 64;        // 16-byte K loads per key row and lane
  constexpr int kDB = kD / 16;        // 16-channel blocks of O
  // m, what the exponents are taken relative to, is the running maximum less kAbove. Any m gives the same
  // weights; with kAbove those of fp16 reach up to 2^14, and one is rounded to within 2^-39 of the
  // largest instead of 2^-25 (many tokens under 2^-25 beside a heavy one would lose all of theirs).
  // bf16 has fp32's range.
  constexpr float kAbove = kF16 ? 14.f : 0.f;
  typedef Half<kF16> E;
  __shared__ float s_o[kWaves][kRows][kD + 4];
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row16 = lane & 15, g = lane >> 4;
  const int page = 1 << c.log_page;
  const int units = row_blocks * c.kv_heads;
  const Place place = kMode == kOneEach ? place_of(c, s, sp, units, wg)
                      : is_few ? Place{0, 1, 0, 0}
                      : kByWave ? Place{wg * kWaves + wave, static_cast<int64_t>(s.batch) * units, 0, 0}
                                : find_share<kPart>(c, s, sp, units, wg);
  int64_t at = place.from;
  const int64_t end = place.to;
  if (at >= end) return;
  const int64_t range0 = at;
  int b = __builtin_amdgcn_readfirstlane(place.seq);
  int64_t seq0 = place.before;   // where sequence b's units begin
  const int all_rows = is_few ? few.rows : io.tokens * io.group;
  const int step = kByWave && !is_few ? kTile : kQuad;   // tokens between two tiles of a wave

  while (at < end) {
    if constexpr (kByWave) b = static_cast<int>(at / units);
    const int len = is_few ? few.tokens : __builtin_amdgcn_readfirstlane(seq_tokens(c, s, b));
    const bool too_long = !is_few && (s.lengths[b] < 0 || s.lengths[b] > len);
    const int nq = quads_of(len), cost = nq + sp.unit_cost;
    if constexpr (kByWave) seq0 = static_cast<int64_t>(b) * units;
    const int unit = static_cast<int>(kByWave ? at - seq0 : (at - seq0) / cost);
    const int64_t unit0 = seq0 + static_cast<int64_t>(unit) * cost;
    const int64_t here = at;
    at = kByWave ? at + static_cast<int64_t>(sp.workgroups) * kWaves : min(end, unit0 + cost);
    int qa = kByWave ? 0 : max(static_cast<int>(here - unit0) - sp.unit_cost, 0);
    int qb = kByWave ? nq : static_cast<int>(at - unit0) - sp.unit_cost;
    if (!kByWave && sp.slots == nullptr) {
      qb = here > unit0 ? 0 : nq;   // another workgroup's, or all of it
      at = unit0 + cost;
    }
    const int b_now = b;
    const bool next_seq = !kByWave && unit + 1 == units && at == unit0 + cost;
    if (next_seq) {
      seq0 = at;
      ++b;
    }
    if (is_few) {
      qa = 0;
      qb = 1;
      at = end;
    }
    if (qb <= qa) continue;
    const int u = is_few ? few.head : unit % c.kv_heads, r_block = is_few ? 0 : (unit / c.kv_heads) * kRows;
    const int* table = is_few ? few.table : s.table + b_now * s.t_st;
    if constexpr (kMode == kShareHeads || kMode == kOneEach) table += u * s.t_sh;
    const int seen0 = is_few ? len : len - io.tokens + 1;   // keys that the first of the Q tokens sees

    // ---- Q: row r_block + 16 nr + row16, channels 64 j + 16 g + 8 s .. + 8 ----
    u32x4 qf[kNR][2 * kKL];
    int limit[kNR];                          // keys that the row sees
#pragma unroll
    for (int nr = 0; nr < kNR; ++nr) {
      const int r = min(r_block + 16 * nr + row16, all_rows - 1);
      int64_t from = b_now;
      int i = r / io.group, h = u * io.group + r - i * io.group;
      if constexpr (kPart)
        if (is_few) {
          const int row = few.row + r;
          i = row / io.group;
          h = u * io.group + row - i * io.group;
          from = few.first + i / io.tokens;
          i %= io.tokens;
        }
      limit[nr] = is_few ? len : seen0 + i;
      const uint16_t* src = io.q + from * io.q_sb + i * io.q_st + h * io.q_sh + 16 * g;
#pragma unroll
      for (int j = 0; j < kKL; ++j) {
        qf[nr][2 * j] = *reinterpret_cast<const u32x4*>(src + 64 * j);
        qf[nr][2 * j + 1] = *reinterpret_cast<const u32x4*>(src + 64 * j + 8);
      }
    }

    f32x4 o[kNR][kDB];
    float m[kNR], l[kNR];
#pragma unroll
    for (int nr = 0; nr < kNR; ++nr) {
      m[nr] = -INFINITY;
      l[nr] = 0.f;
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[nr][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float unit_scale = 0.f;                  // fp16: O in units of this power of two (0: O is 0)
    bool bad = too_long;

    // Pages of a tile's 16-token groups: lane's K rows lie in group row16 / 4, its V run and
    // scores in group g. Groups behind the last token repeat the last one.
    const int last_group = max(len - 1, 0) & ~15;
    // Ids and scales stay as loaded until they are used: a check here would wait for every load
    // that was issued before.
    struct Ids {
      int k, v;   // page of the lane's K rows, of its V run
    };
    auto ids_of = [&](int tile0) __attribute__((always_inline)) {
      return Ids{table[min(tile0 + 16 * (row16 >> 2), last_group) >> c.log_page],
                 table[min(tile0 + 16 * g, last_group) >> c.log_page]};
    };
    auto in_pool = [&](int id) __attribute__((always_inline)) { return id >= 0 && id < c.pages; };
    auto scale_of = [&](const uint8_t* scales, int id) __attribute__((always_inline)) {
      return static_cast<uint32_t>(scales[static_cast<int64_t>(in_pool(id) ? id : 0) * c.kv_heads + u]);
    };
    u32x4 kr[4][kKL], vr[kDB];
    auto load_k = [&](int id, int tile0) __attribute__((always_inline)) {
      const int pos = min(tile0 + 16 * (row16 >> 2), last_group) & (page - 1);
      const uint8_t* p = c.k + (static_cast<int64_t>(in_pool(id) ? id : 0) * c.kv_heads + u) * page * kD +
                         (pos + (row16 & 3)) * kD + 16 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < kKL; ++j)
          kr[t][j] = *reinterpret_cast<const u32x4*>(p + 4 * t * kD + 64 * j);
    };
    auto load_v = [&](int id, int tile0) __attribute__((always_inline)) {
      const int pos = min(tile0 + 16 * g, last_group) & (page - 1);
      const uint8_t* p = c.v + (static_cast<int64_t>(in_pool(id) ? id : 0) * c.kv_heads + u) * page * kD +
                         row16 * page + pos;
#pragma unroll
      for (int db = 0; db < kDB; ++db) vr[db] = *reinterpret_cast<const u32x4*>(p + 16 * db * page);
    };

    // The codes of a tile are loaded one step ahead, K's as soon as the scores have used the
    // last ones and V's after the product; their page ids one step before that, the scales with K.
    int tile0 = is_few ? (few.from + wave) * kTile : kByWave ? 0 : (qa * kWaves + wave) * kTile;
    const int tile_end = min(is_few ? few.to * kTile : qb * kQuad, len);
    if (tile0 < tile_end) {
      Ids now = ids_of(tile0), next = ids_of(tile0 + step);
      load_k(now.k, tile0);
      uint32_t ks = scale_of(c.ks, now.v), vs = scale_of(c.vs, now.v);
      load_v(now.v, tile0);
      for (; tile0 < tile_end; tile0 += step) {
        bad |= !in_pool(now.v);                          // the g groups are all of the tile's
        const int next0 = tile0 + step;
        const bool more = next0 < tile_end;
        const Ids after = ids_of(next0 + step);
        // ---- Sᵀ ----
        f32x4 sc_t[kNR][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int nr = 0; nr < kNR; ++nr) sc_t[nr][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < kKL; ++j) {
            const u32x4 a0 = widen8<kF16>(kr[t][j][0], kr[t][j][1], 1.f);
            const u32x4 a1 = widen8<kF16>(kr[t][j][2], kr[t][j][3], 1.f);
#pragma unroll
            for (int nr = 0; nr < kNR; ++nr) {
              sc_t[nr][t] = E::mfma(a0, qf[nr][2 * j], sc_t[nr][t]);
              sc_t[nr][t] = E::mfma(a1, qf[nr][2 * j + 1], sc_t[nr][t]);
            }
          }
        }
        const float k_scale = e8m0_scale(max(ks, kLeastScaleByte)) * scale_log2;
        uint32_t top = max(vs, kLeastScaleByte);
        float v_scale = e8m0_scale(top);
        if (more) {
          load_k(next.k, next0);
          ks = scale_of(c.ks, next.v);
          vs = scale_of(c.vs, next.v);
        }

        // ---- fp16: V's scales relative to the tile's largest one ----
        // A code keeps all its bits down to 2^-15 of that (2^-9, the least, is then 2^-24); what a page is
        // further below goes into its tokens' weights instead, which the lane holds with their V.
        float weight = 1.f;
        bool apart = false;
        if (kF16) {
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
          // within what fp16 values ask for (2^-32 .. 2^16), so that no rescaling overflows
          const float tile_scale = e8m0_scale(min(max(top, 127u - 32u), 127u + 16u));
          if (tile_scale != unit_scale) {   // wave-uniform
            const float f = unit_scale == 0.f ? 1.f : unit_scale / tile_scale;
#pragma unroll
            for (int nr = 0; nr < kNR; ++nr)
#pragma unroll
              for (int db = 0; db < kDB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nr][db][i] *= f;
            unit_scale = tile_scale;
          }
          const float below = v_scale / tile_scale;
          v_scale = fmaxf(below, 0x1p-15f);
          weight = fminf(below * 0x1p15f, 1.f);
          apart = __any(weight < 1.f);
        }

        // ---- softmax: scores times K's scale, running maximum in exp2 units ----
        const bool masked = tile0 + kTile > seen0;
        u32x4 pb[kNR][2];
#pragma unroll
        for (int nr = 0; nr < kNR; ++nr) {
          float mx = -INFINITY;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x = sc_t[nr][t][i] * k_scale;
              if (masked && tile0 + 16 * g + 4 * t + i >= limit[nr]) x = -INFINITY;
              sc_t[nr][t][i] = x;
              mx = fmaxf(mx, x);
            }
          mx = max_quad_rows(mx);
          const bool grow = mx - m[nr] > kAbove;
          if (__any(grow)) {
            const float m_new = grow ? below<kF16>(mx, kAbove) : m[nr];
            const float corr = m[nr] == m_new ? 1.f : __builtin_amdgcn_exp2f(m[nr] - m_new);
            m[nr] = m_new;
            l[nr] *= corr;
#pragma unroll
            for (int db = 0; db < kDB; ++db)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[nr][db][i] *= corr;
          }
          const float m_safe = m[nr] == -INFINITY ? 0.f : m[nr];  // a row that sees nothing yet
          float p[16], sum = 0.f;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              p[4 * t + i] = __builtin_amdgcn_exp2f(sc_t[nr][t][i] - m_safe);
              sum += p[4 * t + i];
            }
          l[nr] += sum;                     // of this lane's keys; joined after the last tile
          if (apart) {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] *= weight;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) pb[nr][h][i] = E::pack(p[8 * h + 2 * i], p[8 * h + 2 * i + 1]);
        }

        // ---- V: tail bytes to zero ----
        if (tile0 + kTile > len) {
          const int n = len - (tile0 + 16 * g);
#pragma unroll
          for (int db = 0; db < kDB; ++db)
#pragma unroll
            for (int w = 0; w < 4; ++w) vr[db][w] &= first_bytes(n - 4 * w);
        }
        // ---- Oᵀ += Vᵀ Pᵀ ----
        bool nans = false;
        if (masked && io.tokens > 1) {
          // a NaN of a token that only some rows see must not reach the others (0 NaN = NaN)
#pragma unroll
          for (int db = 0; db < kDB; ++db)
#pragma unroll
            for (int w = 0; w < 4; ++w) nans |= nan_bytes(vr[db][w]) != 0;
          nans = __any(nans);
        }
        if (nans) {
          u32x4 seen[kNR][2];
#pragma unroll
          for (int nr = 0; nr < kNR; ++nr)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int key = tile0 + 16 * g + 8 * h + 2 * i;
                seen[nr][h][i] = E::pack(key < limit[nr] ? 1.f : 0.f, key + 1 < limit[nr] ? 1.f : 0.f);
              }
#pragma unroll
          for (int db = 0; db < kDB; ++db) {
            f32x4 hits[kNR];
#pragma unroll
            for (int nr = 0; nr < kNR; ++nr) hits[nr] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t n0 = nan_bytes(vr[db][2 * h]), n1 = nan_bytes(vr[db][2 * h + 1]);
              const u32x4 a = widen8<kF16>(n0, n1, 1.f);
              vr[db][2 * h] &= ~(((n0 >> 3) & 0x01010101u) * 0xffu);
              vr[db][2 * h + 1] &= ~(((n1 >> 3) & 0x01010101u) * 0xffu);
#pragma unroll
              for (int nr = 0; nr < kNR; ++nr) hits[nr] = E::mfma(a, seen[nr][h], hits[nr]);
            }
#pragma unroll
            for (int nr = 0; nr < kNR; ++nr)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (hits[nr][i] > 0.f) o[nr][db][i] = __uint_as_float(0x7fc00000u);
          }
        }
#pragma unroll
        for (int db = 0; db < kDB; ++db)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32x4 a = widen8<kF16>(vr[db][2 * h], vr[db][2 * h + 1], v_scale);
#pragma unroll
            for (int nr = 0; nr < kNR; ++nr) o[nr][db] = E::mfma(a, pb[nr][h], o[nr][db]);
          }
        if (more) load_v(next.v, next0);
        now = next;
        next = after;
      }
    }

    // ---- join the four waves ----
    if (__any(bad)) {
      if (lane == 0) *c.faults = 1;
#pragma unroll
      for (int nr = 0; nr < kNR; ++nr) l[nr] = __uint_as_float(0x7fc00000u);
    }
    if (kByWave && !is_few) {    // nothing to join: the wave's values are the unit's
      const float f = kF16 ? unit_scale : 1.f;
#pragma unroll
      for (int nr = 0; nr < kNR; ++nr) {
        const float sum = sum_quad_rows(l[nr]);
        const int row = r_block + 16 * nr + row16;
        if (row >= all_rows) continue;
        const int i = row / io.group, h = u * io.group + row - i * io.group;
        float* dst = part + ((static_cast<int64_t>(b_now) * io.tokens + i) * c.kv_heads * io.group + h) * (kD + 4);
#pragma unroll
        for (int db = 0; db < kDB; ++db) {
          f32x4 x = o[nr][db];
          if (kF16)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] *= f;
          *reinterpret_cast<f32x4*>(dst + 16 * db + 4 * g) = x;
        }
        if (g == 0) {
          dst[kD] = m[nr];
          dst[kD + 1] = sum;
        }
      }
      continue;
    }
    __syncthreads();   // the previous unit's values are read
#pragma unroll
    for (int nr = 0; nr < kNR; ++nr) {
      const float sum = sum_quad_rows(l[nr]);
      if (g == 0) {
        s_m[wave][16 * nr + row16] = m[nr];
        s_l[wave][16 * nr + row16] = sum;
      }
      const float f = kF16 ? unit_scale : 1.f;
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        f32x4 x = o[nr][db];
        if (kF16)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] *= f;
        *reinterpret_cast<f32x4*>(&s_o[wave][16 * nr + row16][16 * db + 4 * g]) = x;
      }
    }
    __syncthreads();
    const bool whole = qa == 0 && qb == nq;
    const int64_t slot = 2 * static_cast<int64_t>(wg) + (here == range0 ? 0 : 1);
    constexpr int kVec = kD / 4;
    for (int e = tid; e < kRows * kVec; e += kThreads) {
      const int r = e / kVec, d = (e % kVec) * 4;
      const int row = r_block + r;
      if (row >= all_rows) break;
      float mw[kWaves], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        mw[w] = s_m[w][r];
        top = fmaxf(top, mw[w]);
      }
      float sum = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        // a wave without a visible key: weight 0. Its sum still carries a fault's NaN; and a NaN of V
        // stays one however small the factor is, so that the result does not depend on the split.
        const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[w] - top);
        sum += s_l[w][r] * f;
        const f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[w][r][d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += x[i] * f;
      }
      if (whole && !kPart) {
        const int i = row / io.group, h = u * io.group + row - i * io.group;
        const float inv = inverse_of(sum, seen0 + i);
        u32x2 y;
        y[0] = E::pack_out(acc[0] * inv, acc[1] * inv);
        y[1] = E::pack_out(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<u32x2*>(io.out + b_now * io.o_sb + i * io.o_st + h * io.o_sh + d) = y;
        if (io.lse != nullptr && d == 0)
          io.lse[(static_cast<int64_t>(b_now) * io.tokens + i) * c.kv_heads * io.group + h] =
              sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
      } else {
        const int i = row / io.group, h = u * io.group + row - i * io.group;
        float* dst = is_few ? few.slot + static_cast<int64_t>(r) * (kD + 4)
            : kPart && whole
            ? part + ((static_cast<int64_t>(b_now) * io.tokens + i) * c.kv_heads * io.group + h) * (kD + 4)
            : sp.slots + (slot * kRows + r) * (kD + 4);
        *reinterpret_cast<f32x4*>(dst + d) = acc;
        if (d == 0) {
          dst[kD] = top;
          dst[kD + 1] = sum;
        }
      }
    }
  }
}

// ---- host ----

// How vdn_cache_attention cuts its work: rows of a row block, and whether units are split.
struct UnitPlan {
  int block, row_blocks;
  bool split;
  Split sp;             // slots to be set by the caller
  int64_t slot_bytes;   // of a split's slots
};
UnitPlan plan_units(int batch, int width, int log_page, int64_t rows, int kv_heads, int head_dim, int block);

// Row blocks of 32 for more than 16 rows (cache_attn.hip).
int rows_of_block(int rows, int head_dim);

}  // namespace units
}  // namespace vdn

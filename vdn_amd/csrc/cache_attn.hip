// Attention of each sequence's newest tokens over the 8-bit key/value cache (kv_cache.h).
//
//   out[b, i, h] = sum_{j < len_b - Q + 1 + i} softmax_j(scale q[b, i, h] . k[j, u]) v[j, u]
//
// for the Q newest tokens of sequence b (their K/V are in the cache already), u = h / G. Every
// K/V head has Q G query rows against all its cached tokens: a few rows, so reading the codes
// bounds it, 2 D bytes per token and K/V head. One token against 131072, 56 heads on 8 x 128: 268 MB in
// 45 us (6 TB/s, as a large read), 64 sequences of 512 - 8192, 40 heads: 368 MB in 72 (5.1: units that
// start and end inside a workgroup's range), and 5 - 6 us of the join.
//
// A wave takes 64 tokens at a time, straight from memory into registers (no LDS, no barrier):
//   Sᵀ[key][row] = K Qᵀ on 16x16x32 MFMAs of 16-bit values. A lane's 16-byte load holds 16
//     channels of one key, i.e. two channel steps; row r of Sᵀ tile t is key 16 (r / 4) + 4 t +
//     r % 4, so that lane (row, g = lane / 16) ends up with the scores of keys 16 g .. 16 g + 15.
//   Oᵀ += Vᵀ Pᵀ: those are the keys of one 16-byte load of a channel row of the transposed V
//     page, and Pᵀ's operand layout, so P stays in registers too.
// E4M3 codes widen to 16 bits exactly. K's scale multiplies the scores, in fp32 (a lane's 16 keys
// lie in one page). V's goes into the widening: bf16 holds every code's value; for fp16 it is
// taken relative to the tile's largest one, and O is kept in units of that. P is rounded to 16 bits,
// the MFMA's operand; its sum keeps fp32.
//
// Each 16 or 32 rows read and widen all codes of their K/V head again. For the few rows of a decode step
// that is one reading; many queries (a piece of a prompt behind cached tokens) pay for it in VALU work: 256
// behind 8192 tokens, 40 heads on 8 x 128, 40 row blocks: 119 us, VALU busy 54% and MFMA 15% of the
// time, where the products alone ask for 33.
//
// Work: a quad is 256 tokens (one tile for each of a workgroup's 4 waves) of one (sequence, row
// block, K/V head) unit. The quads of all units in order, and one more for each unit, are shared
// out evenly over the workgroups, which find their share from the lengths on the device (with
// tables of up to kWholeQuads a unit stays whole, for the workgroup in whose share it starts). A
// workgroup that holds a unit's every quad writes its output; else it leaves maximum, sum and O in
// a slot, and a second kernel joins a unit's slots in order (no atomics: the same call gives the
// same bits).
#include "cache_units.h"

#include <algorithm>

namespace vdn {
namespace {

using namespace units;

// kPart: nothing is divided by the sums; a whole unit's rows go to `part` as a slot's do.
template <int kD, int kNR, bool kF16, bool kPart>
__global__ void __launch_bounds__(kThreads, workgroups_per_cu(kD, 16 * kNR))
cache_attn_kernel(KvCache c, Queries io, Lengths s, Split sp, int row_blocks, float scale_log2, float* part) {
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
  const int wg = blockIdx.x;
  const Place place = find_share(c, s, sp, units, wg);
  int64_t at = place.from;
  const int64_t end = place.to;
  if (at >= end) return;
  const int64_t range0 = at;
  int b = __builtin_amdgcn_readfirstlane(place.seq);
  int64_t seq0 = place.before;   // where sequence b's units begin
  const int all_rows = io.tokens * io.group;

  while (at < end) {
    const int len = __builtin_amdgcn_readfirstlane(seq_tokens(c, s, b));
    const bool too_long = s.lengths[b] < 0 || s.lengths[b] > len;
    const int nq = quads_of(len), cost = nq + sp.unit_cost;
    const int unit = static_cast<int>((at - seq0) / cost);
    const int64_t unit0 = seq0 + static_cast<int64_t>(unit) * cost;
    const int64_t here = at;
    at = min(end, unit0 + cost);
    int qa = max(static_cast<int>(here - unit0) - sp.unit_cost, 0);
    int qb = static_cast<int>(at - unit0) - sp.unit_cost;
    if (sp.slots == nullptr) {
      qb = here > unit0 ? 0 : nq;   // another workgroup's, or all of it
      at = unit0 + cost;
    }
    const int b_now = b;
    const bool next_seq = unit + 1 == units && at == unit0 + cost;
    if (next_seq) {
      seq0 = at;
      ++b;
    }
    if (qb <= qa) continue;
    const int u = unit % c.kv_heads, r_block = (unit / c.kv_heads) * kRows;
    const int* table = s.table + b_now * s.t_st + u * s.t_sh;
    const int seen0 = len - io.tokens + 1;   // keys that the first of the Q tokens sees

    // ---- Q: row r_block + 16 nr + row16, channels 64 j + 16 g + 8 s .. + 8 ----
    u32x4 qf[kNR][2 * kKL];
    int limit[kNR];                          // keys that the row sees
#pragma unroll
    for (int nr = 0; nr < kNR; ++nr) {
      const int r = min(r_block + 16 * nr + row16, all_rows - 1);
      const int i = r / io.group, h = u * io.group + r - i * io.group;
      limit[nr] = seen0 + i;
      const uint16_t* src = io.q + b_now * io.q_sb + i * io.q_st + h * io.q_sh + 16 * g;
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
    int tile0 = (qa * kWaves + wave) * kTile;
    const int tile_end = min(qb * kQuad, len);
    if (tile0 < tile_end) {
      Ids now = ids_of(tile0), next = ids_of(tile0 + kQuad);
      load_k(now.k, tile0);
      uint32_t ks = scale_of(c.ks, now.v), vs = scale_of(c.vs, now.v);
      load_v(now.v, tile0);
      for (; tile0 < tile_end; tile0 += kQuad) {
        bad |= !in_pool(now.v);                          // the g groups are all of the tile's
        const int next0 = tile0 + kQuad;
        const bool more = next0 < tile_end;
        const Ids after = ids_of(next0 + kQuad);
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
          mx = max_quad_rows(mx) - kAbove;
          if (__any(mx > m[nr])) {
            const float m_new = fmaxf(m[nr], mx);
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
        float* dst = kPart && whole
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

// Joins the slots of every unit that more than one workgroup worked on: a workgroup per row of a
// unit, kD / 4 lanes for the channels, the others take slots in turn. One wave where rows are many
// (units then have few slots), four where they are few (and have many).
template <int kD, int kNR, bool kF16, int kJoinWaves>
__global__ void __launch_bounds__(64 * kJoinWaves)
cache_join_kernel(KvCache c, Queries io, Lengths s, Split sp, int row_blocks) {
  constexpr int kRows = 16 * kNR;
  constexpr int kVec = kD / 4, kLanes = 64 * kJoinWaves / kVec;   // slots at a time
  __shared__ float s_part[kLanes][kD], s_pm[kLanes], s_pl[kLanes];
  const int units = row_blocks * c.kv_heads;
  const int rows = io.tokens * io.group;
  const int b = blockIdx.x / (rows * c.kv_heads);
  const int row = blockIdx.x / c.kv_heads % rows, u = blockIdx.x % c.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63;
  int all = 0, front = 0, own = 0;
  for (int i = lane; i < s.batch; i += 64) {
    const int n = cost_of(sp, seq_tokens(c, s, i));
    all += n;
    if (i < b) front += n;
    if (i == b) own = n;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    all += __shfl_xor(all, d);
    front += __shfl_xor(front, d);
    own += __shfl_xor(own, d);
  }
  const int64_t total = static_cast<int64_t>(all) * units;
  const int64_t start = static_cast<int64_t>(front) * units +
                        static_cast<int64_t>((row / kRows) * c.kv_heads + u) * own;
  const int n_wg = static_cast<int>(min(total, static_cast<int64_t>(sp.workgroups)));
  const int64_t w0 = share_of(total, n_wg, start + sp.unit_cost);
  const int64_t w1 = share_of(total, n_wg, start + own - 1);
  if (w0 == w1) return;   // written by its one workgroup
  const int second = start > share_from(total, n_wg, static_cast<int>(w0)) ? 1 : 0;
  const int d = (tid % kVec) * 4, part = tid / kVec;
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 8;   // slots in flight
  for (int64_t w = w0 + part; w <= w1; w += kLanes * kAhead) {
    f32x4 x[kAhead];
    float m[kAhead], l[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t wa = min(w + a * kLanes, w1);
      const int64_t slot = 2 * wa + (wa == w0 ? second : 0);
      const float* src = sp.slots + (slot * kRows + row % kRows) * (kD + 4);
      x[a] = *reinterpret_cast<const f32x4*>(src + d);
      m[a] = src[kD];
      l[a] = src[kD + 1];
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (w + a * kLanes > w1) break;
      const float m_new = fmaxf(top, m[a]);
      const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - m_new);
      const float f1 = m[a] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[a] - m_new);
      sum = sum * f0 + l[a] * f1;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = acc[i] * f0 + x[a][i] * f1;
      top = m_new;
    }
  }
  if (kLanes > 1) {
    *reinterpret_cast<f32x4*>(&s_part[part][d]) = acc;
    if (d == 0) {
      s_pm[part] = top;
      s_pl[part] = sum;
    }
    __syncthreads();
    if (part != 0) return;
    top = -INFINITY;
    for (int i = 0; i < kLanes; ++i) top = fmaxf(top, s_pm[i]);
    sum = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < kLanes; ++i) {
      const float f = s_pm[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_pm[i] - top);
      sum += s_pl[i] * f;
      const f32x4 x = *reinterpret_cast<const f32x4*>(&s_part[i][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += x[j] * f;
    }
  }
  const int i = row / io.group, h = u * io.group + row - i * io.group;
  const float inv = inverse_of(sum, seq_tokens(c, s, b) - io.tokens + 1 + i);
  u32x2 y;
  y[0] = Half<kF16>::pack_out(acc[0] * inv, acc[1] * inv);
  y[1] = Half<kF16>::pack_out(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<u32x2*>(io.out + b * io.o_sb + i * io.o_st + h * io.o_sh + d) = y;
  if (io.lse != nullptr && d == 0)
    io.lse[(static_cast<int64_t>(b) * io.tokens + i) * c.kv_heads * io.group + h] =
        sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace vdn

using namespace vdn;

namespace vdn {
namespace {

// Row blocks of 32 for more than 16 rows: every code is loaded and widened once for both halves.
// With 256 channels 32 rows spill (50.1 us against 50.4 in blocks of 16: 16 sequences of 4096
// tokens, 4 K/V heads, 32 rows), so those stay at 16.
int rows_of_block(int rows, int head_dim) { return rows > 16 && head_dim <= 128 ? 32 : 16; }

// As many workgroups as run at once, fewer if there are not so many quads at all.
int64_t workgroups_of(int64_t most_quads, int head_dim, int block) {
  const int64_t fit = static_cast<int64_t>(workgroups_per_cu(head_dim, block)) * cu_count();
  return std::max<int64_t>(1, std::min(fit, most_quads));
}

}  // namespace

namespace units {

UnitPlan plan_units(int batch, int width, int log_page, int64_t rows, int kv_heads, int head_dim) {
  UnitPlan p;
  p.block = rows_of_block(static_cast<int>(std::min<int64_t>(rows, 32)), head_dim);
  p.row_blocks = static_cast<int>((rows + p.block - 1) / p.block);
  const int64_t unit_quads = ((static_cast<int64_t>(width) << log_page) + kQuad - 1) / kQuad;
  const int64_t all = static_cast<int64_t>(p.row_blocks) * kv_heads * batch;
  p.split = unit_quads > kWholeQuads;
  p.sp = Split{nullptr, static_cast<int>(workgroups_of(all * unit_quads, head_dim, p.block)),
               p.split ? kUnitCost : 0};
  p.slot_bytes = p.split ? 4ll * 2 * p.sp.workgroups * p.block * (head_dim + 4) : 0;
  return p;
}

int launch_partials(const KvCache& c, const Queries& io, const Lengths& s, const UnitPlan& plan, float* whole,
                    int head_dim, int dtype, float scale_log2, hipStream_t stream) {
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.sp.workgroups)), dim3(kThreads), 0, stream, c, io, s,
                       plan.sp, plan.row_blocks, scale_log2, whole);
  };
#define VDN_PART(D, NR) \
  dtype ? launch(cache_attn_kernel<D, NR, true, true>) : launch(cache_attn_kernel<D, NR, false, true>)
  if (head_dim == 64)
    plan.block == 16 ? (VDN_PART(64, 1)) : (VDN_PART(64, 2));
  else if (head_dim == 128)
    plan.block == 16 ? (VDN_PART(128, 1)) : (VDN_PART(128, 2));
  else
    VDN_PART(256, 1);
#undef VDN_PART
  return check_launch("cache partials");
}

}  // namespace units
}  // namespace vdn

VDN_API int vdn_cache_attention_workspace(int tokens, int group, int head_dim, int64_t* bytes) {
  if (bytes == nullptr || tokens <= 0 || group <= 0)
    return set_error(kInvalidArgument, "vdn_cache_attention_workspace: invalid argument");
  const int64_t rows = static_cast<int64_t>(tokens) * group;
  const int block = rows_of_block(static_cast<int>(std::min<int64_t>(rows, 32)), head_dim);
  *bytes = 4ll * 2 * workgroups_per_cu(head_dim, block) * cu_count() * block * (head_dim + 4);
  return kOk;
}

namespace {

int cache_attention(const char* name, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                    const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                    int* faults, int pages, int kv_heads, int page, int head_dim, const int* table,
                    int64_t table_st, int64_t table_sh, int batch, int width, const int* lengths, int tokens,
                    int group, int dtype, float scale, void* out, int64_t o_sb, int64_t o_st, int64_t o_sh,
                    float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const KvCache c{static_cast<uint8_t*>(const_cast<void*>(k_codes)),
                  static_cast<uint8_t*>(const_cast<void*>(k_scales)),
                  static_cast<uint8_t*>(const_cast<void*>(v_codes)),
                  static_cast<uint8_t*>(const_cast<void*>(v_scales)), faults, pages, kv_heads,
                  page > 0 ? 31 - __builtin_clz(static_cast<unsigned>(page)) : 0};
  if (!cache_geometry_ok(c, page, head_dim) || batch < 0 || width <= 0 || tokens <= 0 || group <= 0 ||
      (static_cast<int64_t>(width) << c.log_page) > (1ll << 31) - 1024)
    return set_error(kInvalidArgument,
                     "%s: bad geometry (page a power of two in 16..256, head_dim 64, 128 or 256)", name);
  if (dtype != 0 && dtype != 1)
    return set_error(kInvalidArgument, "%s: dtype must be 0 (bf16) or 1 (fp16)", name);
  if (!(scale > 0.f) || !isfinite(scale)) return set_error(kInvalidArgument, "%s: bad scale", name);
  if (batch == 0) return kOk;
  if (q == nullptr || out == nullptr || c.k == nullptr || c.ks == nullptr || c.v == nullptr ||
      c.vs == nullptr || faults == nullptr || table == nullptr || lengths == nullptr)
    return set_error(kInvalidArgument, "%s: null pointer", name);
  if (!aligned16(q) || !aligned16(out) || !aligned16(c.k) || !aligned16(c.v) || q_sb % 8 || q_st % 8 ||
      q_sh % 8 || o_sb % 8 || o_st % 8 || o_sh % 8)
    return set_error(kInvalidArgument, "%s: codes and rows need 16-byte alignment", name);
  const int64_t rows = static_cast<int64_t>(tokens) * group;
  if (rows * kv_heads * batch * kThreads >= (1ll << 32))
    return set_error(kUnsupported, "%s: too many query rows", name);
  UnitPlan plan = plan_units(batch, width, c.log_page, rows, kv_heads, head_dim);
  const int block = plan.block, row_blocks = plan.row_blocks, workgroups = plan.sp.workgroups;
  const bool split = plan.split;
  if (split) {
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < plan.slot_bytes)
      return set_error(kInvalidArgument, "%s: workspace missing, unaligned or too small", name);
    plan.sp.slots = static_cast<float*>(workspace);
  }
  const Split& sp = plan.sp;
  const int64_t unit_quads = ((static_cast<int64_t>(width) << c.log_page) + kQuad - 1) / kQuad;
  const Queries io{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(out), lse, q_sb, q_st, q_sh,
                   o_sb, o_st, o_sh, tokens, group};
  const Lengths s{table, lengths, table_st, table_sh, batch, width};
  if (batch * (unit_quads + kUnitCost) > (1ll << 31) - 1) return set_error(kUnsupported, "%s: too many tokens", name);
  const int64_t join_rows = rows * kv_heads * batch;
  const auto launch = [&](auto main, auto join1, auto join4) {
    const auto st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(main, dim3(static_cast<unsigned>(workgroups)), dim3(kThreads), 0, st, c, io, s, sp,
                       row_blocks, scale * kLog2e, static_cast<float*>(nullptr));
    if (!split) return;
    const dim3 grid(static_cast<unsigned>(join_rows));
    if (join_rows > 4 * cu_count())
      hipLaunchKernelGGL(join1, grid, dim3(64), 0, st, c, io, s, sp, row_blocks);
    else
      hipLaunchKernelGGL(join4, grid, dim3(256), 0, st, c, io, s, sp, row_blocks);
  };
#define VDN_CACHE(D, NR, F16)                                               \
  launch(cache_attn_kernel<D, NR, F16, false>, cache_join_kernel<D, NR, F16, 1>, \
         cache_join_kernel<D, NR, F16, 4>)
#define VDN_CACHE_D(F16)                                                            \
  head_dim == 64 ? (block == 16 ? VDN_CACHE(64, 1, F16) : VDN_CACHE(64, 2, F16))    \
  : head_dim == 128 ? (block == 16 ? VDN_CACHE(128, 1, F16) : VDN_CACHE(128, 2, F16)) \
                    : VDN_CACHE(256, 1, F16)
  if (dtype == 0)
    VDN_CACHE_D(false);
  else
    VDN_CACHE_D(true);
#undef VDN_CACHE_D
#undef VDN_CACHE
  return check_launch(name);
}

}  // namespace

VDN_API int vdn_cache_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                const void* k_codes, const void* k_scales, const void* v_codes,
                                const void* v_scales, int* faults, int pages, int kv_heads, int page,
                                int head_dim, const int* table, int64_t table_st, int batch,
                                int width, const int* lengths, int tokens, int group, int dtype,
                                float scale, void* out, int64_t o_sb, int64_t o_st, int64_t o_sh,
                                float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  return cache_attention("vdn_cache_attention", q, q_sb, q_st, q_sh, k_codes, k_scales, v_codes, v_scales, faults,
                         pages, kv_heads, page, head_dim, table, table_st, 0, batch, width, lengths, tokens, group,
                         dtype, scale, out, o_sb, o_st, o_sh, lse, workspace, workspace_bytes, stream);
}

VDN_API int vdn_cache_attention_heads(const void* q, int64_t q_sb, int64_t q_sh, const void* k_codes,
                                      const void* k_scales, const void* v_codes, const void* v_scales,
                                      int* faults, int pages, int kv_heads, int page, int head_dim,
                                      const int* tables, int64_t table_sb, int64_t table_sh, int batch, int width,
                                      const int* lengths, int group, int dtype, float scale, void* out,
                                      int64_t o_sb, int64_t o_sh, float* lse, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  return cache_attention("vdn_cache_attention_heads", q, q_sb, 0, q_sh, k_codes, k_scales, v_codes, v_scales,
                         faults, pages, kv_heads, page, head_dim, tables, table_sb, table_sh, batch, width, lengths,
                         1, group, dtype, scale, out, o_sb, 0, o_sh, lse, workspace, workspace_bytes, stream);
}

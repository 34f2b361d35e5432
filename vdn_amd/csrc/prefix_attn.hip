// Attention of sequences that share prefixes in the 8-bit cache (kv_cache.h), each prefix read once for all.
//
//   out[b, i, h] = softmax over the prefix of b (all its tokens) and b's own tail (the tokens
//                  j < len_b - Q + 1 + i) of scale q[b, i, h] . k[j, u], times v[j, u];   u = h / G
//
// The rows (sequence, i, g) of a prefix that share a K/V head are cut into blocks of 128; the host's plan
// cuts the prefix's tokens into pieces, so that all blocks' pieces fill most of the card once. A
// workgroup takes one piece for one block: four waves of 32 rows, tiles of 64 tokens whose codes
// go global -> LDS, double-buffered, and are widened to 16 bits by each wave as it reads them. (128 rows: one
// reading of the codes serves many sequences, and two workgroups of 128 channels fit a CU.)
//   Sᵀ[key][row] = K Qᵀ on 32x32x16 MFMAs; row r of the A operand is key 16 (r / 4 % 2) + 4 (r / 8)
//     + r % 4, so that half h of the wave ends up with the scores of keys 16 h .. 16 h + 15
//   Oᵀ += Vᵀ Pᵀ: those are the keys of one 16-byte read of a channel of the transposed V page, and
//     Pᵀ's operand layout: P stays in registers
// K's scale multiplies the scores in fp32; V's goes into the widening (bf16), or is taken relative to
// the tile's largest one (fp16, as in cache_attn.hip). P is rounded to 16 bits, its sum keeps fp32.
//
// 16 rows or fewer would leave three of the four waves without work: the workgroup takes such a piece with
// the decode kernel's code instead, the waves dividing its tiles. 8 prefixes of 32768 tokens, two sequences
// each, 16 heads on 8: 50 us against 79 with 64 channels, 109 against 113 with 128, 198 against 323 with 256
// (the bytes alone are 45, 90 and 179; decode over repeated tables takes 68, 135 and 258).
//
// Each piece leaves maximum, sum and O of its rows in fp32, other workgroups of the launch, with the decode
// kernel's code, the same of the tails, and a second kernel joins them in order (no atomics: the
// same call gives the same bits).
//
// VALU work bounds it, with the MFMAs beside it and the clock at the power limit: of a wave's 32 rows and
// 64 tokens x 128 channels, 128 conversions and 160 instructions of softmax go with 32 MFMAs (60 and
// 36% of the time busy). 128 sequences behind 65536 tokens, 40 heads on 8 x 128, tails of 16 - 1000: 214 - 231 us by
// card, 0.75 - 0.81 PFLOP/s; a large library product reaches 1.24. Short prefixes are bound by latency: 4 sequences
// behind 500 tokens, 12 heads on 2 x 64: 5.8 us and 3.6 of the join.
#include "cache_units.h"

#include <algorithm>
#include <type_traits>

namespace vdn {
namespace {

constexpr int kRowsOfBlock = 128;
constexpr int kBN = 64;         // tokens of a tile
constexpr int kThreads = 256;
constexpr int kFewRows = 16;    // the plan's pieces of so few rows are whole steps of four tiles

using units::Half;
using units::Lengths;
using units::Queries;
using units::Split;

// The plan's rows (int32 [.., 8]).
struct Item {      // a piece of a prefix for a block of rows
  int prefix;
  int first;       // first sequence of the prefix
  int row, rows;   // first row of the block, rows of the prefix (sequences x Q x G)
  int tile, end;   // tiles of 64 tokens
  int tokens;      // of the prefix
  int slot;        // where the piece's partial results begin: rows in front of them
};
struct Sequence {
  int first;       // first sequence of its prefix
  int item;        // first item of the prefix
  int pieces, blocks;
  int tokens;      // of the prefix
  int slot, rows;  // its first piece's slot, and the rows that every piece has
  int unused;
};

// Partial result of row r of a piece of n rows, K/V head u: [D + 4] floats (O, m, l, two unused). A piece's rows lie
// behind each other for each K/V head in turn, `slot` rows of the pieces in front of it before them.
template <int kD>
__device__ __forceinline__ float* slot_row(float* slots, int64_t slot, int64_t n, int kv_heads, int u, int64_t r) {
  return slots + (slot * kv_heads + n * u + r) * (kD + 4);
}

struct Prefixes {
  const int* table;
  int64_t t_st;
  int width;
};

__device__ __forceinline__ float max_halves(float x) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

// Workgroups on a CU, by registers.
constexpr int per_cu(int head_dim) { return head_dim == 256 ? 1 : 2; }

// 16-byte chunk c of key k's row lies at c ^ swz(k): 16 lanes of an operand read, keys 8 a .. 8 a + 7 and 16
// behind them, then meet all 64 banks once.
template <int kD>
__device__ __forceinline__ int swz(int key) {
  const int far = key >> 4 & 1;
  return kD == 64 ? (key >> 2 & 1) | far << 1 : kD == 128 ? (key >> 1 & 3) | far << 2 : (key & 7) | far << 3;
}

// The item and the K/V head of a workgroup. With a multiple of 8 K/V heads each XCD keeps its own heads: the
// blocks of a piece share an L2.
struct Piece {
  int item, head;
};
__device__ __forceinline__ Piece piece_of(int pid, int n_items, int kv_heads) {
  if (kv_heads % 8) return {pid / kv_heads, pid % kv_heads};
  const int local = pid >> 3;
  return {local % n_items, (pid & 7) + 8 * (local / n_items)};
}

// kBig: pages of at least 64 tokens, a tile lies in one; else its four groups of 16 tokens may
// lie in as many.
template <int kD, bool kF16, bool kBig>
__device__ __forceinline__ void attend_prefix(const KvCache& c, const Queries& io, const Prefixes& pre,
                                              const Item* __restrict__ items, int n_items, float* slots,
                                              float scale_log2, const Piece& piece) {
  constexpr int kDB = kD / 32;            // 32-channel accumulators of O
  constexpr int kChunks = kD / 16;        // 16-byte chunks of a key
  constexpr int kKJ = kD / 32;            // a lane's 16-byte reads of a key
  constexpr int kSegs = kD / 64;          // 1 KB segments of K and of V that a wave loads
  constexpr int kIds = kBig ? 1 : 4;
  constexpr float kAbove = kF16 ? 11.f : 0.f;   // m: the running maximum less kAbove (cache_attn.hip)
  typedef Elem<kF16> E;
  typedef typename E::x8 x8;
  // one array per buffer: the compiler then tells a prefetch into one from reads of the other
  __shared__ __attribute__((aligned(1024))) uint8_t sK0[kBN * kD];
  __shared__ __attribute__((aligned(1024))) uint8_t sK1[kBN * kD];
  __shared__ __attribute__((aligned(1024))) uint8_t sV0[kBN * kD];
  __shared__ __attribute__((aligned(1024))) uint8_t sV1[kBN * kD];

  const int u = piece.head;
  const Item it = items[piece.item];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int page = 1 << c.log_page;
  const int* table = pre.table + it.prefix * pre.t_st;
  const int last_group = (it.tokens - 1) & ~15;
  const int64_t head_bytes = static_cast<int64_t>(page) * kD;

  // A tile's page ids come two tiles ahead, its codes and scales one. They stay as loaded until the
  // next tile: a look at an id would wait for all loads in front of it, the codes' among them.
  struct Ids {
    int at[kIds];
  };
  auto load_ids = [&](int t) __attribute__((always_inline)) {
    Ids ids;
#pragma unroll
    for (int g = 0; g < kIds; ++g)
      ids.at[g] = table[min(min(t * kBN + 16 * g, last_group) >> c.log_page, pre.width - 1)];
    return ids;
  };
  auto uniform = [&](const Ids& loaded) __attribute__((always_inline)) {
    Ids ids;
#pragma unroll
    for (int g = 0; g < kIds; ++g) ids.at[g] = __builtin_amdgcn_readfirstlane(loaded.at[g]);
    return ids;
  };
  auto in_pool = [&](int id) __attribute__((always_inline)) { return id >= 0 && id < c.pages; };
  auto block_of = [&](int id) __attribute__((always_inline)) {
    return static_cast<int64_t>(in_pool(id) ? id : 0) * c.kv_heads + u;
  };

  // ---- a tile's codes to LDS: wave w loads keys 16 w .. + 15, and of V a quarter of the channels (kBig,
  // rows of four 16-token chunks, chunk g of channel d at g ^ (d / 4 % 4)) or group w of all
  // channels (rows of one chunk, a group after the other) ----
  const int k_token = lane / kChunks, k_phys = lane % kChunks;
  uint32_t koff[kSegs], voff[kSegs];
#pragma unroll
  for (int j = 0; j < kSegs; ++j) {
    const int token = j * (64 / kChunks) + k_token;
    koff[j] = static_cast<uint32_t>(token * kD + 16 * (k_phys ^ swz<kD>(16 * wave + token)));
    const int ch = kBig ? (wave * kSegs + j) * 16 + (lane >> 2) : 64 * j + lane;
    voff[j] = static_cast<uint32_t>(ch * page + (kBig ? 16 * ((lane & 3) ^ (ch >> 2 & 3)) : 0));
  }
  auto issue = [&](const Ids& ids, int t, uint8_t* dk, uint8_t* dv) __attribute__((always_inline)) {
    const int64_t block = block_of(kBig ? ids.at[0] : wave == 0 ? ids.at[0] : wave == 1 ? ids.at[kIds > 1 ? 1 : 0]
                                                    : wave == 2 ? ids.at[kIds > 1 ? 2 : 0] : ids.at[kIds - 1]);
    const int pos = (kBig ? t * kBN : min(t * kBN + 16 * wave, last_group)) & (page - 1);
    const auto k = tile_rsrc(c.k + block * head_bytes + (pos + (kBig ? 16 * wave : 0)) * kD);
    const auto v = tile_rsrc(c.v + block * head_bytes + pos);
#pragma unroll
    for (int j = 0; j < kSegs; ++j) {
      load_to_lds16(k, koff[j], 0, dk + (wave * kSegs + j) * 1024);
      load_to_lds16(v, voff[j], 0, dv + (wave * kSegs + j) * 1024);
    }
  };
  // K's and V's scale bytes of the lane's two 16-token groups (16 h of either half of the tile). Loaded by
  // lane, with an offset that the compiler cannot tell to be zero for all: it would make a uniform
  // byte a scalar at once, and wait for it there.
  struct Scales {
    uint32_t k[2], v[2];
  };
  int zero = 0;
  asm volatile("" : "+v"(zero));
  auto scales_of = [&](const Ids& ids) __attribute__((always_inline)) {
    Scales s;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int id = kBig ? ids.at[0] : h ? ids.at[kIds > 1 ? 2 * kt + 1 : 0] : ids.at[kIds > 1 ? 2 * kt : 0];
      const int64_t block = block_of(id);
      if (kBig && kt) {
        s.k[1] = s.k[0];
        s.v[1] = s.v[0];
      } else {
        s.k[kt] = c.ks[block + zero];
        s.v[kt] = c.vs[block + zero];
      }
    }
    return s;
  };

  Ids now = uniform(load_ids(it.tile)), ahead = load_ids(it.tile + 1);
  issue(now, it.tile, sK0, sV0);
  Scales sc = scales_of(now);

  // ---- Q: row w0 + col, channels 32 j + 16 h + 8 s .. + 8 ----
  const int w0 = it.row + 32 * wave;
  const bool live = w0 < it.rows;
  const int heads_rows = io.tokens * io.group;
  x8 qf[kKJ][2];
  {
    const int r = min(w0 + col, it.rows - 1);
    const int seq = r / heads_rows, rest = r - seq * heads_rows;
    const int i = rest / io.group, hd = u * io.group + rest - i * io.group;
    const uint16_t* src = io.q + (static_cast<int64_t>(it.first) + seq) * io.q_sb + i * io.q_st + hd * io.q_sh + 16 * h;
#pragma unroll
    for (int j = 0; j < kKJ; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        qf[j][s] = __builtin_bit_cast(x8, *reinterpret_cast<const u32x4*>(src + 32 * j + 8 * s));
  }

  f32x16 o[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  // m starts finite: a tile whose scores are all -inf then adds nothing instead of inf - inf
  constexpr float kLeast = -3.402823466e38f;
  float m = kLeast, l = 0.f;
  bool far = false;                        // some row's m is beyond kFarScore
  float unit_scale = 0.f;                  // fp16: O in units of this power of two (0: O is 0)
  bool bad = false;
  // With one wave a SIMD half of the registers are accumulation registers, and O stays in them if the
  // rare branches that compute on it hand it back there (causal_attn.hip). An accumulator at a time: all at once
  // pass through 128 registers, and what those spilled was reloaded behind the next tile's codes (8 prefixes
  // of 32768 tokens, two sequences each: 451 us, 337).
  auto keep = [&](int db) __attribute__((always_inline)) {
    if constexpr (per_cu(kD) == 1) asm volatile("" : "+a"(o[db]));
  };
  auto rescale = [&](float f) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      keep(db);
#pragma unroll
      for (int v = 0; v < 16; ++v) o[db][v] *= f;
      keep(db);
    }
  };
  // Where the lane's operands begin in a tile: read j of a key (32 keys further the swizzle is the same),
  // and the channels of its group in either half of the tile.
  const int key_row = 16 * (col >> 2 & 1) + 4 * (col >> 3) + (col & 3);   // key of the lane's A row
  int k_at[kKJ], v_at[2];
#pragma unroll
  for (int j = 0; j < kKJ; ++j) k_at[j] = key_row * kD + 16 * ((2 * j + h) ^ swz<kD>(key_row));
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int g = 2 * kt + h;
    v_at[kt] = kBig ? col * 64 + 16 * (g ^ (col >> 2 & 3)) : (g * kD + col) * 16;
  }

  // The last tile is apart if the prefix ends inside it: the others have no token to hide.
  auto process = [&](int t, auto buf_tag, auto tail_tag) __attribute__((always_inline)) {
    constexpr int kBuf = decltype(buf_tag)::value;
    constexpr bool kTail = decltype(tail_tag)::value;
    const uint8_t* tk = kBuf == 0 ? sK0 : sK1;
    const uint8_t* tv = kBuf == 0 ? sV0 : sV1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's share of the tile is there
    __syncthreads();                                   // all of it, and every wave is done with the other buffer
#pragma unroll
    for (int g = 0; g < kIds; ++g) bad |= !in_pool(now.at[g]);
    const Scales s_now = sc;
    if (t + 1 < it.end) {
      now = uniform(ahead);
      issue(now, t + 1, kBuf == 0 ? sK1 : sK0, kBuf == 0 ? sV1 : sV0);
      sc = scales_of(now);
      ahead = load_ids(t + 2);
    }
    if (!live) return;

    // ---- Sᵀ: kAtOnce operand reads are under way before the first is used, and an operand is widened
    // between the MFMAs of the one before. With 256 channels all of them (323 us; four at once 337) ----
    constexpr int kReads = 2 * kKJ, kAtOnce = kD == 256 ? 16 : kD == 128 && !kF16 ? 8 : 4;
    f32x16 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[kt][v] = 0.f;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int r0 = 0; r0 < kReads; r0 += kAtOnce) {
      u32x4 w[kAtOnce];
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
        const int j = (r0 + r) / 2, kt = (r0 + r) & 1;
        w[r] = *reinterpret_cast<const u32x4*>(tk + k_at[j] + kt * 32 * kD);
      }
      __builtin_amdgcn_sched_barrier(0);
      u32x4 lo = units::widen8<kF16>(w[0][0], w[0][1], 1.f), hi = units::widen8<kF16>(w[0][2], w[0][3], 1.f);
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
        const int j = (r0 + r) / 2, kt = (r0 + r) & 1, n = r + 1 < kAtOnce ? r + 1 : r;
        __builtin_amdgcn_sched_barrier(0);
        s[kt] = E::mfma(__builtin_bit_cast(x8, lo), qf[j][0], s[kt]);
        if (n > r) lo = units::widen8<kF16>(w[n][0], w[n][1], 1.f);
        __builtin_amdgcn_sched_barrier(0);
        s[kt] = E::mfma(__builtin_bit_cast(x8, hi), qf[j][1], s[kt]);
        if (n > r) hi = units::widen8<kF16>(w[n][2], w[n][3], 1.f);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // V's operands, the first ones read while the softmax runs
    constexpr int kVAhead = kD == 256 || (kD == 128 && !kF16) ? 8 : 4;
    u32x4 vw[kVAhead];
    auto read_v = [&](int x) __attribute__((always_inline)) {
      vw[x % kVAhead] = *reinterpret_cast<const u32x4*>(tv + v_at[x / kDB] + x % kDB * 32 * (kBig ? 64 : 16));
    };
#pragma unroll
    for (int x = 0; x < kVAhead; ++x) read_v(x);
    __builtin_amdgcn_sched_barrier(0);

    // ---- V's scales; fp16: relative to the tile's largest one (cache_attn.hip) ----
    float v_scale[2], weight[2] = {1.f, 1.f};
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) v_scale[kt] = e8m0_scale(max(s_now.v[kt], kLeastScaleByte));
    bool apart = false;
    if (kF16) {
      uint32_t top = max(max(s_now.v[0], s_now.v[1]), kLeastScaleByte);
      if (!kBig) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      // within what fp16 values ask for (2^-32 .. 2^16), so that no rescaling overflows
      const float tile_scale = e8m0_scale(min(max(top, 127u - 32u), 127u + 16u));
      if (__any(tile_scale != unit_scale)) {   // wave-uniform
        const float f = unit_scale == 0.f ? 1.f : unit_scale / tile_scale;
        rescale(f);
        unit_scale = tile_scale;
      }
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const float below = v_scale[kt] / tile_scale;
        v_scale[kt] = fmaxf(below, 0x1p-15f);
        weight[kt] = fminf(below * 0x1p15f, 1.f);
        apart |= weight[kt] < 1.f;
      }
      apart = __any(apart);
    }

    // ---- softmax: the scores times K's scale. m follows the running maximum at once, so that the heaviest
    // weight is a power of two and not rounded: outputs within 2.1e-3 relative of 64 bits in bf16, where
    // their own rounding makes 1.7e-3; with an m that may lag by 2^8 it is 2.3e-3, and 4% faster ----
    [[maybe_unused]] const int left = it.tokens - t * kBN;     // tokens of the tile
    if constexpr (kTail) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (32 * kt + 16 * h + v >= left) s[kt][v] = -INFINITY;
    }
    float k_scale[2], mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      k_scale[kt] = e8m0_scale(max(s_now.k[kt], kLeastScaleByte)) * scale_log2;
      float top = s[kt][0];
#pragma unroll
      for (int v = 1; v < 16; ++v) top = fmaxf(top, s[kt][v]);
      mx = fmaxf(mx, top * k_scale[kt]);
    }
    mx = max_halves(mx);
    const bool grow = mx - m > kAbove;
    if (__any(grow)) {
      const float m_new = grow ? below<kF16>(mx, kAbove) : m;
      const float corr = grow ? __builtin_amdgcn_exp2f(m - m_new) : 1.f;
      l *= corr;
      rescale(corr);
      m = m_new;
      far = __any(fabsf(m) > kFarScore && m != kLeast);
    }
    if (__builtin_expect(far, 0)) {
      // m is the rounded product of a score and its scale: a score's own product has to be rounded like it.
      // (Following that costs 1%: 128 sequences behind 65536 tokens, 40 heads on 8 x 128, 199.4 us against 197.7.)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kt][v] *= k_scale[kt];
        k_scale[kt] = 1.f;
      }
    }
    u32x4 pb[2][2];
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        s[kt][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][v], k_scale[kt], -m));
        if constexpr (kTail)     // K's scale times the softmax's may be 0 in fp32, and 0 inf is NaN
          if (32 * kt + 16 * h + v >= left) s[kt][v] = 0.f;
        sum += s[kt][v];
      }
      if (apart) {
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kt][v] *= weight[kt];
      }
#pragma unroll
      for (int v = 0; v < 16; v += 2) pb[kt][v / 8][v % 8 / 2] = Half<kF16>::pack(s[kt][v], s[kt][v + 1]);
    }
    l += sum;   // of this lane's keys; the halves are joined at the end

    // ---- Oᵀ += Vᵀ Pᵀ ----
    __builtin_amdgcn_sched_barrier(0);
    auto widen_v = [&](int x, int half) __attribute__((always_inline)) {
      uint32_t w0 = vw[x % kVAhead][2 * half], w1 = vw[x % kVAhead][2 * half + 1];
      if constexpr (kTail) {     // behind the last token: 0 NaN is NaN
        const int n = left - 16 * (2 * (x / kDB) + h) - 8 * half;
        w0 &= units::first_bytes(n);
        w1 &= units::first_bytes(n - 4);
      }
      return units::widen8<kF16>(w0, w1, v_scale[x / kDB]);
    };
    __builtin_amdgcn_s_setprio(1);
    u32x4 lo = widen_v(0, 0), hi = widen_v(0, 1);
#pragma unroll
    for (int x = 0; x < 2 * kDB; ++x) {
      const int kt = x / kDB, db = x % kDB;
      if (x + kVAhead < 2 * kDB) read_v(x + kVAhead);
      __builtin_amdgcn_sched_barrier(0);
      o[db] = E::mfma(__builtin_bit_cast(x8, lo), __builtin_bit_cast(x8, pb[kt][0]), o[db]);
      if (x + 1 < 2 * kDB) lo = widen_v(x + 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      o[db] = E::mfma(__builtin_bit_cast(x8, hi), __builtin_bit_cast(x8, pb[kt][1]), o[db]);
      if (x + 1 < 2 * kDB) hi = widen_v(x + 1, 1);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto first = std::integral_constant<int, 0>{};
  const auto second = std::integral_constant<int, 1>{};
  const int whole = min(it.end, it.tokens / kBN);      // behind the last tile that is full
  int t = it.tile;
  for (; t + 1 < whole; t += 2) {
    process(t, first, std::false_type{});
    process(t + 1, second, std::false_type{});
  }
  if (t < whole) {
    process(t, first, std::false_type{});
    if (t + 1 < it.end) process(t + 1, second, std::true_type{});
  } else if (t < it.end) {
    process(t, first, std::true_type{});
  }

#pragma unroll
  for (int db = 0; db < kDB; ++db) keep(db);
  l = sum_halves(l);
  if (bad) {
    if (tid == 0) *c.faults = 1;
    l = __uint_as_float(0x7fc00000u);
  }
  if (!live || w0 + col >= it.rows) return;
  float* dst = slot_row<kD>(slots, it.slot, it.rows, c.kv_heads, u, w0 + col);
  const float f = kF16 ? unit_scale : 1.f;
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<f32x4*>(dst + 32 * db + 8 * j + 4 * h) =
          f32x4{o[db][4 * j] * f, o[db][4 * j + 1] * f, o[db][4 * j + 2] * f, o[db][4 * j + 3] * f};
  if (h == 0) {
    dst[kD] = m;
    dst[kD + 1] = l;
  }
}

// The first workgroups of the decode kernel's launch take a piece of a prefix each, the others share the tails. (The
// other way round workgroups that find nothing to share end at once, and the pieces that follow in their
// places are spread unevenly over the CUs: 308 us instead of 236 for 128 sequences behind 65536 tokens.)
template <int kD, bool kF16, bool kBig>
struct PrefixFront {
  static constexpr int kPerCu = per_cu(kD);
  Prefixes pre;
  const Item* items;
  float* slots;
  int n_items, workgroups;
  // true: the workgroup is to take `few` as a unit.
  __device__ __forceinline__ bool run(const KvCache& c, const Queries& io, float scale_log2, int pid,
                                      units::FewRows& few) const {
    const Piece piece = piece_of(pid, n_items, c.kv_heads);
    const Item it = items[piece.item];
    if (it.rows - it.row <= kFewRows) {
      few = {pre.table + it.prefix * pre.t_st, slot_row<kD>(slots, it.slot, it.rows, c.kv_heads, piece.head, it.row),
             it.first, it.row, it.rows - it.row, piece.head, it.tile, it.end, min(it.tokens, pre.width << c.log_page)};
      return true;
    }
    attend_prefix<kD, kF16, kBig>(c, io, pre, items, n_items, slots, scale_log2, piece);
    return false;
  }
};

// Joins a row's partial results: of the prefix's pieces, in order, then of the tail. A workgroup per
// row, kD / 4 lanes for the channels, the others take partial results in turn.
template <int kD, bool kF16, int kWaves>
__global__ void __launch_bounds__(64 * kWaves)
prefix_join_kernel(KvCache c, Queries io, Lengths s, Split sp, int unit_rows, int row_blocks,
                   const Sequence* __restrict__ seqs, float* __restrict__ slots, const float* __restrict__ whole) {
  constexpr int kVec = kD / 4, kLanes = 64 * kWaves / kVec;
  __shared__ float s_part[kLanes][kD], s_pm[kLanes], s_pl[kLanes];
  const int rows = io.tokens * io.group;
  const int b = blockIdx.x / (rows * c.kv_heads);
  const int row = blockIdx.x / c.kv_heads % rows, u = blockIdx.x % c.kv_heads;
  const int i = row / io.group, head = u * io.group + row - i * io.group;
  const int tid = threadIdx.x, lane = tid & 63;
  const Sequence q = seqs[b];

  // ---- the tail's partial results: a whole unit's, or the slots of the workgroups that shared it ----
  int64_t w0 = 0, w1 = 0;
  int second = 0;
  if (sp.slots != nullptr) {
    int all = 0, front = 0, own = 0;
    for (int j = lane; j < s.batch; j += 64) {
      const int n = units::cost_of(sp, units::seq_tokens(c, s, j));
      all += n;
      if (j < b) front += n;
      if (j == b) own = n;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      all += __shfl_xor(all, d);
      front += __shfl_xor(front, d);
      own += __shfl_xor(own, d);
    }
    const int64_t n_units = static_cast<int64_t>(row_blocks) * c.kv_heads;
    const int64_t total = all * n_units;
    const int64_t start = front * n_units + static_cast<int64_t>(row / unit_rows * c.kv_heads + u) * own;
    const int n_wg = units::sharers<true>(sp, total);
    w0 = units::share_of(total, n_wg, start + sp.unit_cost);
    w1 = units::share_of(total, n_wg, start + own - 1);
    second = start > units::share_from(total, n_wg, static_cast<int>(w0)) ? 1 : 0;
  }
  const int64_t r = static_cast<int64_t>(b - q.first) * rows + row;     // row of the prefix
  const int n = q.pieces + static_cast<int>(w1 - w0) + 1;
  const float* first = slot_row<kD>(slots, q.slot, q.rows, c.kv_heads, u, r);
  const int64_t apart = static_cast<int64_t>(q.rows) * c.kv_heads * (kD + 4);
  auto partial = [&](int x) __attribute__((always_inline)) {
    if (x < q.pieces)
      return first + x * apart;
    if (w0 == w1)
      return whole + ((static_cast<int64_t>(b) * io.tokens + i) * c.kv_heads * io.group + head) * (kD + 4);
    const int64_t w = w0 + x - q.pieces;
    return const_cast<const float*>(sp.slots) +
           ((2 * w + (w == w0 ? second : 0)) * unit_rows + row % unit_rows) * (kD + 4);
  };

  const int d = tid % kVec * 4, part = tid / kVec;
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 4;   // partial results in flight
  for (int x0 = part; x0 < n; x0 += kLanes * kAhead) {
    f32x4 x[kAhead];
    float m[kAhead], l[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const float* src = partial(min(x0 + a * kLanes, n - 1));
      x[a] = *reinterpret_cast<const f32x4*>(src + d);
      m[a] = src[kD];
      l[a] = src[kD + 1];
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (x0 + a * kLanes >= n) break;
      const float m_new = fmaxf(top, m[a]);
      const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - m_new);
      const float f1 = m[a] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[a] - m_new);
      sum = sum * f0 + l[a] * f1;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = acc[j] * f0 + x[a][j] * f1;
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
    for (int j = 0; j < kLanes; ++j) top = fmaxf(top, s_pm[j]);
    sum = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < kLanes; ++j) {
      const float f = s_pm[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_pm[j] - top);
      sum += s_pl[j] * f;
      const f32x4 y = *reinterpret_cast<const f32x4*>(&s_part[j][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += y[e] * f;
    }
  }
  const int keys = q.tokens + max(units::seq_tokens(c, s, b) - io.tokens + 1 + i, 0);
  const float inv = units::inverse_of(sum, keys);
  u32x2 y;
  y[0] = Half<kF16>::pack_out(acc[0] * inv, acc[1] * inv);
  y[1] = Half<kF16>::pack_out(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<u32x2*>(io.out + b * io.o_sb + i * io.o_st + head * io.o_sh + d) = y;
  if (io.lse != nullptr && d == 0)
    io.lse[(static_cast<int64_t>(b) * io.tokens + i) * c.kv_heads * io.group + head] =
        sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How the tails' units are shared out beside n pieces of at most piece_tiles tiles. A tile of 128 rows takes
// less than half as long as a quad of 16 (2.0 and 4.5 us with 128 channels). Where the card's other
// places would do for the longest tails that the table can hold, only those are launched: workgroups that find
// nothing to share wait for a place all the same (128 sequences behind 65536 tokens: 235 us, 250).
//
// Short tables leave a workgroup's waves little to share: one quad of 60 tokens keeps one of the four busy, and
// the workgroup's units run one after another. Where units are not split, each wave takes its own when the
// table holds no more than one wave's tile, or when the units outnumber the places. 40 query heads on 8 of 128
// channels: 256 tails of 1 - 60 tokens 34.1 us against 53.2, of 200 - 500 69.3 against 91.2; but 16 of
// 200 - 500 22.8 against 17.2. Tables of four quads and more gain nothing by it (96 tails of 100 - 1000: 46.2, 43.2).
struct TailPlan : units::UnitPlan {
  bool by_wave;
};
TailPlan plan_tails(int batch, int width, int log_page, int64_t rows, int kv_heads, int head_dim, int64_t n,
                    int piece_tiles) {
  TailPlan plan{units::plan_units(batch, width, log_page, rows, kv_heads, head_dim, 16), false};
  Split& sp = plan.sp;
  const int64_t fit = static_cast<int64_t>(per_cu(head_dim)) * cu_count();
  const int64_t n_units = static_cast<int64_t>(batch) * plan.row_blocks * kv_heads;
  plan.by_wave = !plan.split && ((static_cast<int64_t>(width) << log_page) <= units::kTile || n_units > fit);
  if (plan.by_wave) {
    sp.workgroups = static_cast<int>(std::min((n_units + units::kWaves - 1) / units::kWaves, fit));
    return plan;
  }
  sp.workgroups = static_cast<int>(std::min<int64_t>(sp.workgroups, fit));
  sp.few = n > 0 && n < fit ? static_cast<int>(fit - n) : 0;
  sp.beside = 0.45f * piece_tiles;
  const int64_t quads = ((static_cast<int64_t>(width) << log_page) + units::kQuad - 1) / units::kQuad;
  const int64_t most = batch * (quads + sp.unit_cost) * plan.row_blocks * kv_heads;
  if (units::few_suffice(sp, most)) {
    sp.workgroups = std::min(sp.workgroups, sp.few);
    sp.few = 0;
  }
  return plan;
}

// The workspace: the tails' rows, the tails' slots, the pieces' rows.
struct Bytes {
  int64_t row, whole, tails;
};

Bytes workspace_of(int64_t out_rows, int head_dim, const units::UnitPlan& plan) {
  const int64_t row = 4ll * (head_dim + 4);
  return Bytes{row, out_rows * row, plan.slot_bytes};
}

}  // namespace
}  // namespace vdn

using namespace vdn;

VDN_API int vdn_prefix_attention_workspace(int blocks, int batch, int width, int page, int tokens, int group,
                                           int kv_heads, int head_dim, int64_t* bytes) {
  if (bytes == nullptr || blocks < 0 || batch < 0 || width <= 0 || tokens <= 0 || group <= 0 || kv_heads <= 0 ||
      page <= 0)
    return set_error(kInvalidArgument, "vdn_prefix_attention_workspace: invalid argument");
  const int64_t rows = static_cast<int64_t>(tokens) * group;
  const auto plan = plan_tails(batch, width, 31 - __builtin_clz(static_cast<unsigned>(page)), rows, kv_heads, head_dim,
                               0, 0);
  const Bytes b = workspace_of(rows * kv_heads * batch, head_dim, plan);
  *bytes = b.whole + b.tails + b.row * blocks * kRowsOfBlock * kv_heads;
  return kOk;
}

VDN_API int vdn_prefix_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k_codes,
                                 const void* k_scales, const void* v_codes, const void* v_scales, int* faults,
                                 int pages, int kv_heads, int page, int head_dim, const int* prefix_table,
                                 int64_t prefix_table_st, int prefix_width, const int* items, int n_items,
                                 int piece_tiles, const int* sequences, const int* table, int64_t table_st, int batch, int width,
                                 const int* lengths, int tokens, int group, int dtype, float scale, void* out,
                                 int64_t o_sb, int64_t o_st, int64_t o_sh, float* lse, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const char* name = "vdn_prefix_attention";
  const KvCache c{static_cast<uint8_t*>(const_cast<void*>(k_codes)),
                  static_cast<uint8_t*>(const_cast<void*>(k_scales)),
                  static_cast<uint8_t*>(const_cast<void*>(v_codes)),
                  static_cast<uint8_t*>(const_cast<void*>(v_scales)), faults, pages, kv_heads,
                  page > 0 ? 31 - __builtin_clz(static_cast<unsigned>(page)) : 0};
  if (!cache_geometry_ok(c, page, head_dim) || batch < 0 || width <= 0 || tokens <= 0 || group <= 0 || n_items < 0 ||
      piece_tiles < 0 ||
      prefix_width < 0 || (n_items > 0 && prefix_width == 0) ||
      (static_cast<int64_t>(std::max(width, prefix_width)) << c.log_page) > (1ll << 31) - 1024)
    return set_error(kInvalidArgument,
                     "%s: bad geometry (page a power of two in 16..256, head_dim 64, 128 or 256)", name);
  if (dtype != 0 && dtype != 1) return set_error(kInvalidArgument, "%s: dtype must be 0 (bf16) or 1 (fp16)", name);
  if (!(scale > 0.f) || !isfinite(scale)) return set_error(kInvalidArgument, "%s: bad scale", name);
  if (batch == 0) return kOk;
  if (q == nullptr || out == nullptr || c.k == nullptr || c.ks == nullptr || c.v == nullptr || c.vs == nullptr ||
      faults == nullptr || table == nullptr || lengths == nullptr || sequences == nullptr ||
      (n_items > 0 && (items == nullptr || prefix_table == nullptr)))
    return set_error(kInvalidArgument, "%s: null pointer", name);
  if (!aligned16(q) || !aligned16(out) || !aligned16(c.k) || !aligned16(c.v) || !aligned16(items) ||
      !aligned16(sequences) || q_sb % 8 || q_st % 8 || q_sh % 8 || o_sb % 8 || o_st % 8 || o_sh % 8)
    return set_error(kInvalidArgument, "%s: codes, rows and the plan need 16-byte alignment", name);
  const int64_t rows = static_cast<int64_t>(tokens) * group, out_rows = rows * kv_heads * batch;
  if (out_rows * kThreads >= (1ll << 32) || rows * batch > (1ll << 31) - 512 ||
      (static_cast<int64_t>(n_items) * kv_heads + (1 << 16)) * kThreads >= (1ll << 32))
    return set_error(kUnsupported, "%s: too many query rows", name);
  if (static_cast<int64_t>(batch) *
          (((static_cast<int64_t>(width) << c.log_page) + units::kQuad - 1) / units::kQuad + units::kUnitCost) >
      (1ll << 31) - 1)
    return set_error(kUnsupported, "%s: too many tokens", name);
  TailPlan plan = plan_tails(batch, width, c.log_page, rows, kv_heads, head_dim,
                             static_cast<int64_t>(n_items) * kv_heads, piece_tiles);
  const Bytes need = workspace_of(out_rows, head_dim, plan);
  const int64_t left = workspace_bytes - need.whole - need.tails;      // every item has a row at least
  if (workspace == nullptr || !aligned16(workspace) || left < need.row * n_items * kv_heads)
    return set_error(kInvalidArgument, "%s: workspace missing, unaligned or too small", name);
  float* whole = static_cast<float*>(workspace);
  if (plan.split) plan.sp.slots = whole + need.whole / 4;
  float* slots = whole + (need.whole + need.tails) / 4;
  const Queries io{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(out), lse, q_sb, q_st, q_sh, o_sb, o_st,
                   o_sh, tokens, group};
  const Lengths s{table, lengths, table_st, 0, batch, width};
  const Prefixes pre{prefix_table, prefix_table_st, prefix_width};
  const auto st = static_cast<hipStream_t>(stream);
  const float scale_log2 = scale * kLog2e;
  const int n_pieces = n_items * kv_heads;
  const auto launch = [&](auto kernel, auto front) {
    front = {pre, reinterpret_cast<const Item*>(items), slots, n_items, n_pieces};
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(n_pieces + plan.sp.workgroups)), dim3(kThreads), 0, st, c, io,
                       s, plan.sp, plan.row_blocks, scale_log2, whole, front);
  };
#define VDN_PREFIX(D, F16, BIG)                                                                      \
  (plan.by_wave ? launch(units::cache_attn_kernel<D, 1, F16, units::kPartsByWave, PrefixFront<D, F16, BIG>>, \
                         PrefixFront<D, F16, BIG>{})                                                 \
                : launch(units::cache_attn_kernel<D, 1, F16, units::kParts, PrefixFront<D, F16, BIG>>,       \
                         PrefixFront<D, F16, BIG>{}))
#define VDN_PREFIX_D(D)                                                            \
  dtype ? (page >= kBN ? VDN_PREFIX(D, true, true) : VDN_PREFIX(D, true, false))   \
        : (page >= kBN ? VDN_PREFIX(D, false, true) : VDN_PREFIX(D, false, false))
  if (head_dim == 64)
    VDN_PREFIX_D(64);
  else if (head_dim == 128)
    VDN_PREFIX_D(128);
  else
    VDN_PREFIX_D(256);
#undef VDN_PREFIX_D
#undef VDN_PREFIX
  const auto join = [&](auto one, auto four) {
    const dim3 grid(static_cast<unsigned>(out_rows));
    if (out_rows > 4 * cu_count())
      hipLaunchKernelGGL(one, grid, dim3(64), 0, st, c, io, s, plan.sp, plan.block, plan.row_blocks,
                         reinterpret_cast<const Sequence*>(sequences), slots, whole);
    else
      hipLaunchKernelGGL(four, grid, dim3(256), 0, st, c, io, s, plan.sp, plan.block, plan.row_blocks,
                         reinterpret_cast<const Sequence*>(sequences), slots, whole);
  };
#define VDN_JOIN(D) \
  dtype ? join(prefix_join_kernel<D, true, 1>, prefix_join_kernel<D, true, 4>) \
        : join(prefix_join_kernel<D, false, 1>, prefix_join_kernel<D, false, 4>)
  if (head_dim == 64)
    VDN_JOIN(64);
  else if (head_dim == 128)
    VDN_JOIN(128);
  else
    VDN_JOIN(256);
#undef VDN_JOIN
  return check_launch(name);
}

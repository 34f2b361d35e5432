// Writing rows into the 8-bit key/value cache, and reading them back (kv_cache.h).
//
// Both move memory only: a write reads 2 bytes and writes 1 per value, a read the reverse. Prompts of
// 40600 tokens x 8 heads x 128: write 59 us (4.2 TB/s), read 54 with cold codes (4.6); a large copy
// reaches 4.9. One token for each of 64 sequences: write 10 us, latency and V's D cache lines a head. A
// workgroup takes one page of one sequence, one K/V head and one side; a wave tile is 2048 values,
// four 16-byte pieces of 8 values a lane. K's order is that of the rows. V's codes are channel
// major: a lane takes the same 8 channels of 4 consecutive positions and transposes its 4 x 8
// codes in registers, so that it moves 4 bytes of each channel, 16 lanes the 64 of a page row.
//
// Which page a workgroup takes: sequence i brings rows [offsets[i], offsets[i + 1]) and can touch
// at most (rows >> log_page) + 2 pages, so with base_i = (offsets[i] >> log_page) + 2 i the
// slots base_i .. base_{i+1} - 1 are its own, base is increasing, and a wave finds the sequence
// of a slot by comparing 64 bases at a time. No lengths are needed on the host.
#include "kv_cache.h"

#include <type_traits>

namespace vdn {
namespace {

constexpr int kTileValues = 2048;

struct Rows {
  uint16_t* k;
  uint16_t* v;
  int64_t k_st, k_sh, v_st, v_sh;  // token / head strides (elements)
  int count;                       // packed rows
};

struct Seqs {
  const int* table;    // [batch, width] page ids, row stride t_st
  const int* starts;   // [batch] tokens in front of the rows
  const int* offsets;  // [batch + 1] row offsets, or null: one row each
  int64_t t_st;
  int batch, width;
};

// What a workgroup does: rows row .. row + n - 1 are positions lo .. lo + n - 1 of page `index`
// of sequence `seq`. n <= 0: nothing. seq == batch: rows behind the last sequence.
struct Piece {
  int seq, index, lo, n;
  int64_t row;
};

// A workgroup's slot, K/V head and side. The heads of a page's rows lie next to each other in
// memory, so they go to neighbouring workgroups.
struct Item {
  int slot, u;
  bool v;
};

__device__ __forceinline__ Item item_of(const KvCache& c) {
  const int w = blockIdx.x, page = w / (2 * c.kv_heads), rest = w - page * 2 * c.kv_heads;
  return Item{page, rest % c.kv_heads, rest >= c.kv_heads};
}

__device__ __forceinline__ int seq_base(const Seqs& s, int i, int log_page) {
  return (s.offsets[i] >> log_page) + 2 * i;
}

// Whether sequence i, with rows off .. next - 1, is not behind the one before it or not inside the rows.
// (unsigned: a negative number is larger than any)
__device__ __forceinline__ bool bad_offsets(uint32_t off, uint32_t next, int i, uint32_t rows) {
  return off > (i == 0 ? 0u : next) || next > rows;
}

__device__ Piece find_piece(const KvCache& c, const Seqs& s, int rows, int slot) {
  const int log_page = c.log_page;
  Piece p{0, 0, 0, 0, 0};
  int64_t first, end;
  int j = 0, start;
  if (s.offsets == nullptr) {
    p.seq = min(slot, s.batch);
    first = min(slot, rows);
    end = min(slot + 1, rows);
    if (p.seq == s.batch) {
      p.row = first;
      p.n = static_cast<int>(end - first);
      return p;
    }
    start = s.starts[p.seq];
  } else {
    // the last i in [0, batch) with base_i <= slot, or the rows behind the last sequence
    const int lane = threadIdx.x & 63;
    const int behind = s.offsets[s.batch];
    int lo = 0, step = 1;
    while (static_cast<int64_t>(step) * 64 < s.batch) step *= 64;
    if (step > 1) {
      // The search loads only a part of the offsets and may pass over a pair that falls, so the threads
      // of the grid look at one pair each (there are more of them than sequences).
      const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
      if (i < s.batch && bad_offsets(s.offsets[i], s.offsets[i + 1], static_cast<int>(i), rows)) *c.faults = 1;
    }
    for (; step > 1; step /= 64) {
      const int64_t i = lo + static_cast<int64_t>(lane) * step;
      const bool le = i < s.batch && seq_base(s, static_cast<int>(i), log_page) <= slot;
      const int found = __popcll(__ballot(le));
      if (found == 0) {
        *c.faults = 1;
        return p;
      }
      lo += (found - 1) * step;
    }
    // the last round loads what the sequence needs with its base: one memory latency less
    const int i = lo + lane;
    int off = 0, next = 0, from = 0, base = 0;
    if (i < s.batch) {
      off = s.offsets[i];
      next = s.offsets[i + 1];
      from = s.starts[i];
      base = (off >> log_page) + 2 * i;
    }
    // Offsets that fall would name a row twice, and the search would pass sequences over; out of range
    // they name rows that are not there. Either way none of these sequences is followed.
    const bool bad = __ballot(bad_offsets(off, next, i, rows)) != 0;   // 0, 0 behind the last one
    const int found = __popcll(__ballot(i < s.batch && base <= slot));
    const int base_end = (behind >> log_page) + 2 * s.batch;
    int o0, o1;
    if (base_end <= slot) {
      p.seq = s.batch;
      j = slot - base_end;
      start = 0;
      o0 = behind;
      o1 = rows;
    } else if (found > 0 && !bad) {
      p.seq = lo + found - 1;
      j = slot - __builtin_amdgcn_readlane(base, found - 1);
      if (j < 0) return p;
      start = __builtin_amdgcn_readlane(from, found - 1);
      o0 = __builtin_amdgcn_readlane(off, found - 1);
      o1 = __builtin_amdgcn_readlane(next, found - 1);
    } else {
      *c.faults = 1;   // bad offsets, or rows in front of the first sequence
      return p;
    }
    if (o0 < 0 || o1 < o0 || o1 > rows) *c.faults = 1;
    first = min(max(o0, 0), rows);
    end = min(max(o1, 0), rows);
    if (p.seq == s.batch) {
      p.row = first + (static_cast<int64_t>(j) << log_page);
      p.n = static_cast<int>(min(end - p.row, static_cast<int64_t>(1) << log_page));
      return p;
    }
  }
  const int64_t from = max(start, 0), stop = from + end - first;
  const int64_t index = (from >> log_page) + j;
  const int64_t lo = max(from, index << log_page), hi = min(stop, (index + 1) << log_page);
  p.index = start < 0 ? -1 : static_cast<int>(index);   // -1: a fault, no page
  p.lo = static_cast<int>(lo - (index << log_page));
  p.n = end > first ? static_cast<int>(max(hi - lo, static_cast<int64_t>(-1))) : 0;
  p.row = first + lo - from;
  return p;
}

template <bool kF16>
__device__ __forceinline__ float widen(uint32_t bits) {
  return kF16 ? f16_bits_to_f32(static_cast<uint16_t>(bits)) : __uint_as_float(bits << 16);
}

// Codes of eight finite 16-bit values (low half first) for the scale s = 2^e.
template <bool kF16>
__device__ __forceinline__ u32x2 codes8(const u32x4& w, float s) {
  if constexpr (!kF16) {
    return e4m3x8_bf16(w, s);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    u32x2 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = w[2 * h], hi = w[2 * h + 1];
      s16x2_t r = {0, 0};
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, lo), s, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, hi), s, true);
      out[h] = __builtin_bit_cast(uint32_t, r);
    }
    return out;
  }
}

// The same for any values. A nonfinite one gives the NaN code; bf16 values over 1.875 * 2^127 count
// as that, so that their code (at most 240 at the largest scale 2^120) stands for a finite number.
template <bool kF16>
__device__ u32x2 codes8_any(const u32x4& w, float s) {
  constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
  u32x2 out = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t b = j ? w[i] >> 16 : w[i] & 0xffffu;
      x[j] = widen<kF16>(b);
      if (!kF16) x[j] = fminf(fmaxf(x[j], -0x1.ep127f), 0x1.ep127f);
      if ((b & 0x7fffu) >= kInf) x[j] = __uint_as_float(0x7fc00000u);
    }
    s16x2_t r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x[0], x[1], s, false);
    out[i >> 1] |= (static_cast<uint32_t>(__builtin_bit_cast(uint32_t, r)) & 0xffffu) << (16 * (i & 1));
  }
  return out;
}

// Four held codes for a scale 2^up larger: rounded once more.
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float up) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return e4m3x4_scaled(lo[0], lo[1], hi[0], hi[1], up);
}

// Piece j (0..3) of tile `t` of a page for this lane: its position in the page and its first
// channel. V: positions 4 a + j of up to 64 positions x 32 channels (the page's own 16 or 32
// positions x 128 or 64).
struct Spot {
  int pos, ch;
};

template <int kD, bool kV>
__device__ __forceinline__ Spot spot(int t, int j, int lane, int log_page) {
  if (!kV) {
    const int piece = t * 256 + j * 64 + lane;
    return Spot{piece / (kD / 8), piece % (kD / 8) * 8};
  }
  const int log_a = min(log_page - 2, 4);             // runs of 4 positions: 2^log_a a tile
  const int groups = 64 >> log_a;                     // 8-channel groups a tile
  const int across = max(kD / 8 / groups, 1);         // tiles side by side
  const int a = lane & ((1 << log_a) - 1), cg = lane >> log_a;
  return Spot{((t / across) << (log_a + 2)) + 4 * a + j, (t % across * groups + cg) * 8};
}

// kTiles wave tiles per wave; the workgroup's waves hold the whole page. (A page of 16 positions
// and 64 channels is half a tile: the lanes behind it have a position or channel outside.)
template <int kD, int kTiles, bool kF16, bool kV>
__device__ __forceinline__ void write_page(const KvCache& c, const Rows& rows, const Seqs& s,
                                           const Piece& p, int u) {
  __shared__ uint32_t s_mag[2][16];
  const int tid = threadIdx.x, lane = tid & 63, threads = blockDim.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = threads >> 6;
  const int page = 1 << c.log_page;
  const int64_t st = kV ? rows.v_st : rows.k_st;
  const uint16_t* src = (kV ? rows.v + u * rows.v_sh : rows.k + u * rows.k_sh) + p.row * st;
  const int end = p.lo + p.n;

  // ---- the new rows (on their way before the page is looked up), and their largest finite
  // magnitude (16-bit ones order as integers) ----
  u32x4 w[kTiles][4];
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Spot at = spot<kD, kV>(t * waves + wave, j, lane, c.log_page);
      w[t][j] = u32x4{0, 0, 0, 0};
      if (at.pos >= p.lo && at.pos < end && at.ch < kD)
        w[t][j] = *reinterpret_cast<const u32x4*>(src + (at.pos - p.lo) * st + at.ch);
    }
  const int id = cache_page(c, s.table + p.seq * s.t_st, p.index, s.width);
  if (id < 0) return;
  const int64_t block = static_cast<int64_t>(id) * c.kv_heads + u;
  uint8_t* codes = (kV ? c.v : c.k) + block * page * kD;
  uint8_t* scale = (kV ? c.vs : c.ks) + block;
  const uint32_t held = p.lo > 0 ? max(static_cast<uint32_t>(*scale), kLeastScaleByte) : 0u;
  constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
  u16x2 pair = {0, 0};
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) pair = __builtin_elementwise_max(pair, mag8_bf16(w[t][j]));
  auto page_max = [&](uint32_t x, uint32_t* shared) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), d)));
    if (waves > 1) {
      if (lane == 0) shared[wave] = x;
      __syncthreads();
      for (int i = 0; i < waves; ++i) x = max(x, shared[i]);
    }
    return x;
  };
  uint32_t mag = page_max(max(pair[0], pair[1]), s_mag[0]);
  // a nonfinite value, or one that is clamped, sends the page to the careful conversion
  const bool plain = mag < (kF16 ? kInf : 0x7f70u);
  if (mag >= kInf) {
    mag = 0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t lo = w[t][j][i] & 0x7fffu, hi = (w[t][j][i] >> 16) & 0x7fffu;
          mag = max(mag, lo < kInf ? lo : 0u);
          mag = max(mag, hi < kInf ? hi : 0u);
        }
    mag = page_max(mag, s_mag[1]);
  }
  uint32_t byte = cache_scale_byte(widen<kF16>(mag));

  // ---- a page that holds tokens keeps the larger scale ----
  if (p.lo > 0) {
    if (byte > held) {
      // every 16-byte run with a held token; positions from lo on are overwritten or unused
      const float up = __uint_as_float(min(byte - held + 127u, 254u) << 23);
      const int runs = kV ? kD * (page / 16) : p.lo * (kD / 16);
      for (int i = tid; i < runs; i += threads) {
        if (kV && (i % (page / 16)) * 16 >= p.lo) continue;
        u32x4* at = reinterpret_cast<u32x4*>(codes) + i;
        u32x4 x = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = rescale4(x[j], up);
        *at = x;
      }
      __syncthreads();  // the new codes may lie in the same runs
    } else {
      byte = held;
    }
  }
  if (waves > 1) __syncthreads();  // every wave has read the held scale
  if (tid == 0) *scale = static_cast<uint8_t>(byte);
  const float sf = e8m0_scale(byte);

  // ---- codes of the new rows ----
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    u32x2 out[4];
    if (plain) {
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = codes8<kF16>(w[t][j], sf);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = codes8_any<kF16>(w[t][j], sf);
    }
    const Spot at = spot<kD, kV>(t * waves + wave, 0, lane, c.log_page);
    if (!kV) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Spot to = spot<kD, kV>(t * waves + wave, j, lane, c.log_page);
        if (to.pos >= p.lo && to.pos < end) *reinterpret_cast<u32x2*>(codes + to.pos * kD + to.ch) = out[j];
      }
    } else if (at.ch < kD && at.pos + 4 > p.lo && at.pos < end) {
      const bool whole = at.pos >= p.lo && at.pos + 4 <= end;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t word = 0;   // channel at.ch + i, 4 positions
#pragma unroll
        for (int j = 0; j < 4; ++j) word |= (out[j][i >> 2] >> (8 * (i & 3)) & 0xffu) << (8 * j);
        uint8_t* to = codes + (at.ch + i) * page + at.pos;
        if (whole) {
          *reinterpret_cast<uint32_t*>(to) = word;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at.pos + j >= p.lo && at.pos + j < end) to[j] = static_cast<uint8_t>(word >> (8 * j));
        }
      }
    }
  }
}

template <int kD, int kTiles, bool kF16>
__global__ void __launch_bounds__(1024) cache_write_kernel(KvCache c, Rows rows, Seqs s) {
  const Item item = item_of(c);
  const Piece p = find_piece(c, s, rows.count, item.slot);
  if (p.n <= 0 || p.seq >= s.batch) return;
  if (item.v)
    write_page<kD, kTiles, kF16, true>(c, rows, s, p, item.u);
  else
    write_page<kD, kTiles, kF16, false>(c, rows, s, p, item.u);
}

// Two values of the codes in the low two bytes, as packed 16-bit numbers. fp16 saturates at its
// largest value (a value next to it may have been rounded up to 65536); NaN stays NaN.
template <bool kF16>
__device__ __forceinline__ uint32_t values2(uint32_t codes, float scale) {
  if (!kF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
  const auto f = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  float a = f[0] * scale, b = f[1] * scale;
  if (fabsf(a) > 65504.f) a = copysignf(65504.f, a);
  if (fabsf(b) > 65504.f) b = copysignf(65504.f, b);
  return f32_to_f16_bits(a) | static_cast<uint32_t>(f32_to_f16_bits(b)) << 16;
}

template <int kD, int kTiles, bool kF16, bool kV>
__device__ __forceinline__ void read_page(const KvCache& c, const Rows& rows, const Piece& p, int id,
                                          int u, uint32_t fill) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int page = 1 << c.log_page;
  const int64_t block = static_cast<int64_t>(max(id, 0)) * c.kv_heads + u;
  const uint8_t* codes = (kV ? c.v : c.k) + block * page * kD;
  const float sf = e8m0_scale(max(static_cast<uint32_t>((kV ? c.vs : c.ks)[block]), kLeastScaleByte));
  const int64_t st = kV ? rows.v_st : rows.k_st;
  uint16_t* dst = (kV ? rows.v + u * rows.v_sh : rows.k + u * rows.k_sh) + p.row * st;
  const int end = p.lo + p.n;
  // all codes first: V as [channel] words of 4 positions, K as rows
  uint32_t w[kTiles][8];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    if (kV) {
      const Spot at = spot<kD, kV>(t * waves + wave, 0, lane, c.log_page);
      const bool any = at.ch < kD && at.pos + 4 > p.lo && at.pos < end;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[t][i] = any ? *reinterpret_cast<const uint32_t*>(codes + (at.ch + i) * page + at.pos) : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Spot at = spot<kD, kV>(t * waves + wave, j, lane, c.log_page);
        u32x2 x = {0, 0};
        if (at.pos >= p.lo && at.pos < end) x = *reinterpret_cast<const u32x2*>(codes + at.pos * kD + at.ch);
        w[t][2 * j] = x[0];
        w[t][2 * j + 1] = x[1];
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Spot at = spot<kD, kV>(t * waves + wave, j, lane, c.log_page);
      if (at.pos < p.lo || at.pos >= end || at.ch >= kD) continue;
      uint32_t x[2];
      if (kV) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[h] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[h] |= (w[t][4 * h + i] >> (8 * j) & 0xffu) << (8 * i);
        }
      } else {
        x[0] = w[t][2 * j];
        x[1] = w[t][2 * j + 1];
      }
      u32x4 out{values2<kF16>(x[0], sf), values2<kF16>(x[0] >> 16, sf), values2<kF16>(x[1], sf),
                values2<kF16>(x[1] >> 16, sf)};
      if (id < 0) out = u32x4{fill, fill, fill, fill};
      *reinterpret_cast<u32x4*>(dst + (at.pos - p.lo) * st + at.ch) = out;
    }
}

template <int kD, int kTiles, bool kF16>
__global__ void __launch_bounds__(1024) cache_read_kernel(KvCache c, Rows rows, Seqs s) {
  const Item item = item_of(c);
  const Piece p = find_piece(c, s, rows.count, item.slot);
  if (p.n <= 0) return;
  const bool behind = p.seq >= s.batch;
  const int id = behind ? -1 : cache_page(c, s.table + p.seq * s.t_st, p.index, s.width);
  // no such page: NaN; rows behind the last sequence: zeros
  const uint32_t fill = behind ? 0u : kF16 ? 0x7e007e00u : 0x7fc07fc0u;
  if (item.v)
    read_page<kD, kTiles, kF16, true>(c, rows, p, id, item.u, fill);
  else
    read_page<kD, kTiles, kF16, false>(c, rows, p, id, item.u, fill);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks and launch shared by both directions.
template <bool kWrite>
int move_rows(const char* name, const KvCache& c, int page, Rows rows, Seqs s, int head_dim, int dtype,
              void* stream) {
  if (!cache_geometry_ok(c, page, head_dim) || rows.count < 0 || s.batch < 0 || s.width < 0)
    return set_error(kInvalidArgument,
                     "%s: bad geometry (page a power of two in 16..256, head_dim 64, 128 or 256)", name);
  if (dtype != 0 && dtype != 1)
    return set_error(kInvalidArgument, "%s: dtype must be 0 (bf16) or 1 (fp16)", name);
  if (rows.count == 0 || (kWrite && s.batch == 0)) return kOk;
  if (c.k == nullptr || c.ks == nullptr || c.v == nullptr || c.vs == nullptr || c.faults == nullptr ||
      rows.k == nullptr || rows.v == nullptr ||
      (s.batch > 0 && (s.starts == nullptr || (s.table == nullptr && s.width > 0))))
    return set_error(kInvalidArgument, "%s: null pointer", name);
  if (!aligned16(c.k) || !aligned16(c.v) || !aligned16(rows.k) || !aligned16(rows.v) || rows.k_st % 8 ||
      rows.k_sh % 8 || rows.v_st % 8 || rows.v_sh % 8)
    return set_error(kInvalidArgument, "%s: codes and rows need 16-byte alignment", name);
  // slots: every sequence's pages, and those of the rows behind the last one
  const int64_t slots = s.offsets == nullptr
                            ? (kWrite ? s.batch : static_cast<int64_t>(max(s.batch, rows.count)))
                            : (rows.count >> c.log_page) + 2 * static_cast<int64_t>(s.batch) + (kWrite ? 0 : 1);
  // waves that hold a page: one tile each, two where that would take over 16 waves
  const int tiles = (page * head_dim + kTileValues - 1) / kTileValues;
  const int waves = tiles > 16 ? 16 : tiles;
  const int64_t workgroups = slots * 2 * c.kv_heads;
  if (workgroups * 64 * waves >= (1ll << 32))
    return set_error(kUnsupported, "%s: too many pages or heads", name);
  const dim3 grid(static_cast<unsigned>(workgroups));
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, static_cast<hipStream_t>(stream), c, rows, s);
  };
#define VDN_MOVE(D, F16)                                                                            \
  (kWrite ? (tiles > 16 ? launch(cache_write_kernel<D, 2, F16>) : launch(cache_write_kernel<D, 1, F16>)) \
          : (tiles > 16 ? launch(cache_read_kernel<D, 2, F16>) : launch(cache_read_kernel<D, 1, F16>)))
  if (dtype == 0)
    head_dim == 64 ? VDN_MOVE(64, false) : head_dim == 128 ? VDN_MOVE(128, false) : VDN_MOVE(256, false);
  else
    head_dim == 64 ? VDN_MOVE(64, true) : head_dim == 128 ? VDN_MOVE(128, true) : VDN_MOVE(256, true);
#undef VDN_MOVE
  return check_launch(name);
}

KvCache cache_of(void* k, void* ks, void* v, void* vs, int* faults, int pages, int kv_heads, int page) {
  return KvCache{static_cast<uint8_t*>(k), static_cast<uint8_t*>(ks), static_cast<uint8_t*>(v),
                 static_cast<uint8_t*>(vs), faults, pages, kv_heads,
                 page > 0 ? 31 - __builtin_clz(static_cast<unsigned>(page)) : 0};
}

}  // namespace
}  // namespace vdn

using namespace vdn;

VDN_API int vdn_cache_write(void* k_codes, void* k_scales, void* v_codes, void* v_scales, int* faults,
                            int pages, int kv_heads, int page, int head_dim, const int* table,
                            int64_t table_st, int batch, int width, const int* starts,
                            const int* offsets, const void* key, int64_t k_st, int64_t k_sh,
                            const void* value, int64_t v_st, int64_t v_sh, int rows, int dtype,
                            void* stream) {
  return move_rows<true>(
      "vdn_cache_write", cache_of(k_codes, k_scales, v_codes, v_scales, faults, pages, kv_heads, page), page,
      Rows{static_cast<uint16_t*>(const_cast<void*>(key)), static_cast<uint16_t*>(const_cast<void*>(value)),
           k_st, k_sh, v_st, v_sh, rows},
      Seqs{table, starts, offsets, table_st, batch, width}, head_dim, dtype, stream);
}

VDN_API int vdn_cache_read(const void* k_codes, const void* k_scales, const void* v_codes,
                           const void* v_scales, int* faults, int pages, int kv_heads, int page,
                           int head_dim, const int* table, int64_t table_st, int batch, int width,
                           const int* starts, const int* offsets, void* key, int64_t k_st,
                           int64_t k_sh, void* value, int64_t v_st, int64_t v_sh, int rows,
                           int dtype, void* stream) {
  return move_rows<false>(
      "vdn_cache_read",
      cache_of(const_cast<void*>(k_codes), const_cast<void*>(k_scales), const_cast<void*>(v_codes),
               const_cast<void*>(v_scales), faults, pages, kv_heads, page),
      page, Rows{static_cast<uint16_t*>(key), static_cast<uint16_t*>(value), k_st, k_sh, v_st, v_sh, rows},
      Seqs{table, starts, offsets, table_st, batch, width}, head_dim, dtype, stream);
}

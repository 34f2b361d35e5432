// Writing rows into the 8-bit key/value cache, and reading them back (kv_cache.h).
//
// Both move memory only: a write reads 2 bytes and writes 1 per value, a read the reverse. A
// workgroup takes one page of one sequence, one K/V head and one side. Rows are 16-bit and token
// major; V goes through LDS to change to the cache's channel-major order and back.
//
// Which page a workgroup takes: sequence i brings rows [offsets[i], offsets[i + 1]) and can touch
// at most (rows >> log_page) + 2 pages, so with base_i = (offsets[i] >> log_page) + 2 i the
// slots base_i .. base_{i+1} - 1 are its own, base is increasing, and a wave finds the sequence
// of a slot by comparing 64 bases at a time. No lengths are needed on the host.
#include "kv_cache.h"

#include <type_traits>

namespace vdn {
namespace {

constexpr int kThreads = 256;

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

__device__ __forceinline__ int seq_base(const Seqs& s, int i, int log_page) {
  return (s.offsets[i] >> log_page) + 2 * i;
}

__device__ Piece find_piece(const KvCache& c, const Seqs& s, int rows, int slot) {
  const int log_page = c.log_page;
  Piece p{0, 0, 0, 0, 0};
  int64_t first, end;
  int j = 0;
  if (s.offsets == nullptr) {
    p.seq = slot;
    first = min(slot, rows);
    end = min(slot + 1, rows);
    if (slot >= s.batch) return p.seq = s.batch, p.row = first, p.n = static_cast<int>(end - first), p;
  } else {
    // the last i in [0, batch] with base_i <= slot
    const int lane = threadIdx.x & 63;
    int lo = 0, step = 1;
    while (static_cast<int64_t>(step) * 64 < s.batch + 1) step *= 64;
    for (; step >= 1; step /= 64) {
      const int64_t i = lo + static_cast<int64_t>(lane) * step;
      const bool le = i <= s.batch && seq_base(s, static_cast<int>(i), log_page) <= slot;
      const int found = __popcll(__ballot(le));
      if (found == 0) return p;
      lo += (found - 1) * step;
    }
    p.seq = min(lo, s.batch);
    j = slot - seq_base(s, p.seq, log_page);
    if (j < 0) return p;
    const int o0 = s.offsets[p.seq], o1 = p.seq == s.batch ? rows : s.offsets[p.seq + 1];
    if (o0 < 0 || o1 < o0 || o1 > rows) *c.faults = 1;
    first = min(max(o0, 0), rows);
    end = min(max(o1, 0), rows);
    if (p.seq == s.batch) {
      p.row = first + (static_cast<int64_t>(j) << log_page);
      p.n = static_cast<int>(min(end - p.row, static_cast<int64_t>(1) << log_page));
      return p;
    }
  }
  const int64_t start = max(s.starts[p.seq], 0), stop = start + end - first;
  const int64_t index = (start >> log_page) + j;
  const int64_t lo = max(start, index << log_page), hi = min(stop, (index + 1) << log_page);
  p.index = s.starts[p.seq] < 0 ? -1 : static_cast<int>(index);   // -1: a fault, no page
  p.lo = static_cast<int>(lo - (index << log_page));
  p.n = end > first ? static_cast<int>(max(hi - lo, static_cast<int64_t>(-1))) : 0;
  p.row = first + lo - start;
  return p;
}

template <bool kF16>
__device__ __forceinline__ float widen(uint32_t bits) {
  return kF16 ? f16_bits_to_f32(static_cast<uint16_t>(bits)) : __uint_as_float(bits << 16);
}

// Codes of two 16-bit values (low half first) in the low two bytes. A nonfinite value gives
// the NaN code; bf16 values over 1.875 * 2^127 count as that, so that their code (at most 240 at
// the largest scale 2^120) stands for a finite number.
template <bool kF16>
__device__ __forceinline__ uint32_t codes2(uint32_t w, float scale) {
  constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
  float x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t b = i ? w >> 16 : w & 0xffffu;
    x[i] = widen<kF16>(b);
    if (!kF16) x[i] = fminf(fmaxf(x[i], -0x1.ep127f), 0x1.ep127f);
    if ((b & 0x7fffu) >= kInf) x[i] = __uint_as_float(0x7fc00000u);
  }
  s16x2_t r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x[0], x[1], scale, false);
  return static_cast<uint32_t>(__builtin_bit_cast(uint32_t, r)) & 0xffffu;
}

// Four held codes for a scale 2^up larger: rounded once more.
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float up) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return e4m3x4_scaled(lo[0], lo[1], hi[0], hi[1], up);
}

template <int kD, bool kF16>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(KvCache c, Rows rows, Seqs s) {
  constexpr int kChunks = kD / 8;             // 8-value pieces of a row
  constexpr int kStep = kThreads / kChunks;   // rows of a pass
  const int page = 1 << c.log_page, pitch = page + 4;
  extern __shared__ uint8_t tile[];           // V: [kD][pitch]
  __shared__ uint32_t s_mag[kThreads / 64];
  const Piece p = find_piece(c, s, rows.count, blockIdx.x);
  if (p.n <= 0 || p.seq >= s.batch) return;
  const int u = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.z != 0;
  const int id = cache_page(c, s.table + p.seq * s.t_st, p.index, s.width);
  if (id < 0) return;
  const int64_t block = static_cast<int64_t>(id) * c.kv_heads + u;
  uint8_t* codes = (is_v ? c.v : c.k) + block * page * kD;
  uint8_t* scale = (is_v ? c.vs : c.ks) + block;
  const int64_t st = is_v ? rows.v_st : rows.k_st;
  const uint16_t* src = (is_v ? rows.v + u * rows.v_sh : rows.k + u * rows.k_sh) + p.row * st;
  const int ch = tid % kChunks, r0 = tid / kChunks;

  // ---- largest finite magnitude of the new rows (16-bit magnitudes order as integers) ----
  constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
  uint32_t mag = 0;
  for (int r = r0; r < p.n; r += kStep) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(src + r * st + 8 * ch);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
      if (lo < kInf) mag = max(mag, lo);
      if (hi < kInf) mag = max(mag, hi);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) mag = max(mag, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mag), d)));
  if ((tid & 63) == 0) s_mag[tid >> 6] = mag;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) mag = max(mag, s_mag[i]);
  uint32_t byte = cache_scale_byte(widen<kF16>(mag));

  // ---- a page that holds tokens keeps the larger scale ----
  if (p.lo > 0) {
    const uint32_t held = max(static_cast<uint32_t>(*scale), kLeastScaleByte);
    if (byte > held) {
      // every 16-byte run with a held token; positions from lo on are overwritten or unused
      const float up = __uint_as_float(min(byte - held + 127u, 254u) << 23);
      const int runs = is_v ? kD * (page / 16) : p.lo * (kD / 16);
      for (int i = tid; i < runs; i += kThreads) {
        if (is_v && (i % (page / 16)) * 16 >= p.lo) continue;
        u32x4* at = reinterpret_cast<u32x4*>(codes) + i;
        u32x4 w = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = rescale4(w[j], up);
        *at = w;
      }
    } else {
      byte = held;
    }
  }
  __syncthreads();  // held codes are rewritten, and every thread has read the held scale
  if (tid == 0) *scale = static_cast<uint8_t>(byte);
  const float sf = e8m0_scale(byte);

  // ---- codes of the new rows ----
  for (int r = r0; r < p.n; r += kStep) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(src + r * st + 8 * ch);
    u32x2 out;
    out[0] = codes2<kF16>(w[0], sf) | codes2<kF16>(w[1], sf) << 16;
    out[1] = codes2<kF16>(w[2], sf) | codes2<kF16>(w[3], sf) << 16;
    if (!is_v) {
      *reinterpret_cast<u32x2*>(codes + (p.lo + r) * kD + 8 * ch) = out;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        tile[(8 * ch + i) * pitch + p.lo + r] = static_cast<uint8_t>(out[i >> 2] >> (8 * (i & 3)));
    }
  }
  if (!is_v) return;
  __syncthreads();
  // rows of 4 positions; a run that holds other positions too goes byte by byte
  const int words = page / 4;
  for (int i = tid; i < kD * words; i += kThreads) {
    const int d = i / words, at = (i % words) * 4;
    if (at + 4 <= p.lo || at >= p.lo + p.n) continue;
    const uint8_t* from = tile + d * pitch + at;
    uint8_t* to = codes + d * page + at;
    if (at >= p.lo && at + 4 <= p.lo + p.n) {
      *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
    } else {
      for (int b = 0; b < 4; ++b)
        if (at + b >= p.lo && at + b < p.lo + p.n) to[b] = from[b];
    }
  }
}

// Two values of the codes in the low two bytes, as packed 16-bit numbers. fp16 saturates at its
// largest value (a value next to it may have been rounded up to 65536); NaN stays NaN.
template <bool kF16>
__device__ __forceinline__ uint32_t values2(uint32_t codes, float scale) {
  const auto f = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  float a = f[0] * scale, b = f[1] * scale;
  if (!kF16) return pack_bf16x2(a, b);
  if (fabsf(a) > 65504.f) a = copysignf(65504.f, a);
  if (fabsf(b) > 65504.f) b = copysignf(65504.f, b);
  return f32_to_f16_bits(a) | static_cast<uint32_t>(f32_to_f16_bits(b)) << 16;
}

template <int kD, bool kF16>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(KvCache c, Rows rows, Seqs s) {
  constexpr int kChunks = kD / 8;
  constexpr int kStep = kThreads / kChunks;
  const int page = 1 << c.log_page, pitch = page + 4;
  extern __shared__ uint8_t tile[];
  const Piece p = find_piece(c, s, rows.count, blockIdx.x);
  if (p.n <= 0) return;
  const int u = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.z != 0;
  const int64_t st = is_v ? rows.v_st : rows.k_st;
  uint16_t* dst = (is_v ? rows.v + u * rows.v_sh : rows.k + u * rows.k_sh) + p.row * st;
  const int ch = tid % kChunks, r0 = tid / kChunks;
  const bool behind = p.seq >= s.batch;
  const int id = behind ? -1 : cache_page(c, s.table + p.seq * s.t_st, p.index, s.width);
  if (id < 0) {  // no such page: NaN; rows behind the last sequence: zeros
    const uint32_t fill = behind ? 0u : kF16 ? 0x7e007e00u : 0x7fc07fc0u;
    for (int r = r0; r < p.n; r += kStep)
      *reinterpret_cast<u32x4*>(dst + r * st + 8 * ch) = u32x4{fill, fill, fill, fill};
    return;
  }
  const int64_t block = static_cast<int64_t>(id) * c.kv_heads + u;
  const uint8_t* codes = (is_v ? c.v : c.k) + block * page * kD;
  const float sf = e8m0_scale(max(static_cast<uint32_t>((is_v ? c.vs : c.ks)[block]), kLeastScaleByte));
  if (is_v) {
    const int runs = page / 16;
    for (int i = tid; i < kD * runs; i += kThreads) {
      const int d = i / runs, at = (i % runs) * 16;
      if (at + 16 <= p.lo || at >= p.lo + p.n) continue;
      const u32x4 w = *reinterpret_cast<const u32x4*>(codes + d * page + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(tile + d * pitch + at + 4 * j) = w[j];
    }
    __syncthreads();
  }
  for (int r = r0; r < p.n; r += kStep) {
    u32x2 w;
    if (!is_v) {
      w = *reinterpret_cast<const u32x2*>(codes + (p.lo + r) * kD + 8 * ch);
    } else {
      w = u32x2{0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2] |= static_cast<uint32_t>(tile[(8 * ch + i) * pitch + p.lo + r]) << (8 * (i & 3));
    }
    const u32x4 out{values2<kF16>(w[0], sf), values2<kF16>(w[0] >> 16, sf),
                    values2<kF16>(w[1], sf), values2<kF16>(w[1] >> 16, sf)};
    *reinterpret_cast<u32x4*>(dst + r * st + 8 * ch) = out;
  }
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
  if (slots > (1ll << 31) - 1 || c.kv_heads > 65535)
    return set_error(kUnsupported, "%s: too many pages or heads", name);
  const dim3 grid(static_cast<unsigned>(slots), static_cast<unsigned>(c.kv_heads), 2);
  const size_t lds = static_cast<size_t>(head_dim) * (page + 4);
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, static_cast<hipStream_t>(stream), c, rows, s);
  };
#define VDN_MOVE(D, F16) \
  (kWrite ? launch(cache_write_kernel<D, F16>) : launch(cache_read_kernel<D, F16>))
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

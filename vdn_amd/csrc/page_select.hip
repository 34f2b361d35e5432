// Mean keys of the 8-bit cache's pages, and the pages that a query's attention is limited to by them.
//
// Means (vdn_cache_means): mean[p, u] = sum over the page's tokens of K, / n, rounded once to bf16.
// E4M3 values are multiples of 2^-9 up to 448, so 64 of them add up exactly in fp32: a lane's share of any
// page. The lanes' sums meet in fp64. Reading the codes bounds it: 34 MB of 8 prompts of 2048 - 8192 tokens x 8 x
// 128 in 5.2 us (in part from the cache in front of HBM). A wave has a page and head to itself: no barrier.
//
// Selection (vdn_cache_select): score(b, i, u, p) = max over the G query heads h of K/V head u of
// q[b, i, h] . mean[p, u], in fp64: the products of 16-bit values are exact there and their sum nearly,
// so that the order of two pages does not hang on the order of a sum. A page of the first or the last
// ones counts as the largest, NaN as +inf. Of equal scores the page in front wins. Then a workgroup per
// (b, i, u) takes the `count` best: by each page's rank, or where they are many by bins and the
// ranks in the last one. Latency and the conversions to fp64 bound it: 64 sequences of up to 128 pages, 40 heads
// on 8 x 128: 12.0 us; 8192 pages, 56 heads on 8: 10.3 for the scores and 8.8 for the taking.
#include "kv_cache.h"

#include "attn_tiles.h"

#include <algorithm>
#include <type_traits>

namespace vdn {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kAloneThreads = 512;   // of a selection whose pages one workgroup scores
constexpr int kTakeThreads = 1024;   // of one from scored pages

struct Spans {
  const int* table;    // [batch, width], row stride t_st
  const int* starts;   // [batch]
  const int* lengths;  // [batch]
  int64_t t_st;
  int batch, width;
};

__device__ __forceinline__ int most_tokens(const KvCache& c, int width) {
  return static_cast<int>(min(static_cast<int64_t>(width) << c.log_page, (1ll << 31) - 1));
}

// Pages first .. first + n - 1 of sequence b; a bad length or start raises the fault word, and none
// of its pages is followed.
struct Span {
  int first, n, tokens;
};

__device__ __forceinline__ Span span_of(const KvCache& c, const Spans& s, int b) {
  const int start = s.starts[b], len = s.lengths[b];
  if (start < 0 || len < 0 || len > most_tokens(c, s.width)) {
    *c.faults = 1;
    return Span{0, 0, 0};
  }
  const int first = start >> c.log_page, end = (len + (1 << c.log_page) - 1) >> c.log_page;
  return Span{first, start < len ? end - first : 0, len};
}

template <int kD>
__global__ void __launch_bounds__(kThreads) page_means_kernel(KvCache c, Spans s, uint16_t* means) {
  constexpr int kChunks = kD / 16;          // lanes of a token's row
  constexpr int kRows = 64 / kChunks;       // tokens at a time
  constexpr int kCh = kD / 64;              // channels that a lane finishes
  __shared__ float s_part[kWaves][kRows][kD];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int page = 1 << c.log_page;

  // Pages of all sequences in order, 64 strips of sequences at a time.
  const int strip = (s.batch + 63) / 64;
  const int b0 = min(lane * strip, s.batch), b1 = min(b0 + strip, s.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += span_of(c, s, b).n;
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t other = __shfl_up(incl, d);
    incl += lane >= d ? other : 0;
  }
  const int64_t total = __shfl(incl, 63) * c.kv_heads;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kWaves;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + wave; item < total; item += stride) {
    const int64_t at = item / c.kv_heads;
    const int u = static_cast<int>(item - at * c.kv_heads);
    const int owner = __popcll(__ballot(incl <= at));
    int64_t before = __shfl(incl - mine, owner);
    int b = __builtin_amdgcn_readlane(b0, owner);
    Span span = span_of(c, s, b);
    while (at - before >= span.n) {
      before += span.n;
      span = span_of(c, s, ++b);
    }
    const int index = span.first + static_cast<int>(at - before);
    const int id = cache_page(c, s.table + b * s.t_st, index, s.width);
    if (id < 0) continue;
    const int n = min(page, span.tokens - (index << c.log_page));
    const int64_t block = static_cast<int64_t>(id) * c.kv_heads + u;
    const uint8_t* codes = c.k + block * page * kD + lane * 16;
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.f;
    for (int t = 0; t < n; t += 4 * kRows) {
      u32x4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = t + j * kRows + lane / kChunks;
        w[j] = u32x4{0, 0, 0, 0};
        if (row < n) w[j] = *reinterpret_cast<const u32x4*>(codes + static_cast<int64_t>(t + j * kRows) * kD);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j][i], false);
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j][i], true);
          sum[4 * i] += lo[0];
          sum[4 * i + 1] += lo[1];
          sum[4 * i + 2] += hi[0];
          sum[4 * i + 3] += hi[1];
        }
    }
    const double factor = static_cast<double>(e8m0_scale(max(static_cast<uint32_t>(c.ks[block]), kLeastScaleByte)));
    float* part = s_part[wave][lane / kChunks] + lane % kChunks * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(part + 4 * i) = f32x4{sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    double total_of[kCh];
#pragma unroll
    for (int i = 0; i < kCh; ++i) total_of[i] = 0.0;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < kCh; ++i) total_of[i] += static_cast<double>(s_part[wave][r][lane * kCh + i]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // fp64 quotients of sums under 2^26 units by at most 256 are closer to a bf16 tie than fp32 could tell
    // only where they are that tie; fp32 in between rounds to odd, so that the result is rounded once
    uint16_t out[kCh];
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
      const double x = total_of[i] / n * factor;
      float f = static_cast<float>(x);
      uint32_t bits = __float_as_uint(f);
      if (static_cast<double>(f) != x && isfinite(f)) {
        // toward zero, then the last bit set
        if (fabs(static_cast<double>(f)) > fabs(x)) --bits;
        bits |= 1;
      }
      out[i] = f32_to_bf16_bits(__uint_as_float(bits));
    }
    uint16_t* dst = means + block * kD + lane * kCh;
    if constexpr (kCh == 1)
      *dst = out[0];
    else
#pragma unroll
      for (int i = 0; i < kCh; i += 2)
        *reinterpret_cast<uint32_t*>(dst + i) = out[i] | static_cast<uint32_t>(out[i + 1]) << 16;
  }
}

// ---------------------------------------------------------------------- selection ----

struct Select {
  const uint16_t* q;
  const uint16_t* means;
  const int* table;
  const int* lengths;
  int* pages;               // [batch, tokens, kv_heads, count]
  int* seen;                // [batch, tokens]
  unsigned long long* keys; // [units, width], or null: in LDS
  int64_t q_sb, q_st, q_sh, t_st;
  int batch, width, tokens, group, count, first, last;
};

// What unit (b, i, u) sees: its number of pages (-1: a fault) and tokens.
struct Sight {
  int have, tokens;
};

__device__ __forceinline__ Sight sight_of(const KvCache& c, const Select& s, int b, int i) {
  const int len = s.lengths[b];
  if (len < 0 || len > most_tokens(c, s.width)) return Sight{-1, -1};
  const int sees = max(len - s.tokens + 1 + i, 0);
  return Sight{(sees + (1 << c.log_page) - 1) >> c.log_page, sees};
}

// A score's bits in rising order; NaN counts as +inf.
__device__ __forceinline__ unsigned long long key_of(double x) {
  const long long b = __double_as_longlong(x + 0.0);   // -0 becomes 0
  return static_cast<unsigned long long>(b) ^ (b < 0 ? ~0ull : 1ull << 63);
}

constexpr unsigned long long kAlways = ~0ull;

// Keys of pages tile .. tile + 15 of a unit: lane's page is tile + lane % 16 (every quarter of the wave gets
// them). An MFMA has four blocks of 4 query rows (A) x 4 pages (B) x 4 channels: lane 16 k + 4 b + i holds row
// i, or page 4 b + i, and channel k D / 4 + s at step s; the product of row i and page j of block b comes
// to lane 16 i + 4 b + j. Four rows a time waste less of the group than an MFMA of 16 rows: 5 rows of 128
// channels take 1024 cycles of the pipe for 16 pages instead of 2048.
template <int kD, bool kF16>
__device__ unsigned long long tile_keys(const KvCache& c, const Select& s, const int* row, int u, int tile,
                                        int have, const uint16_t* q, int64_t q_sh) {
  constexpr int kRun = kD / 4;      // channels of a lane
  const int lane = threadIdx.x & 63, k = lane >> 4;
  const int at = tile + (lane & 15);
  const int id = at < have ? row[at] : 0;
  const bool there = id >= 0 && id < c.pages;
  if (!there) *c.faults = 1;
  u32x4 w[kRun / 8];
  const uint16_t* m = s.means + (static_cast<int64_t>(there ? id : 0) * c.kv_heads + u) * kD + k * kRun;
#pragma unroll
  for (int j = 0; j < kRun / 8; ++j) w[j] = *reinterpret_cast<const u32x4*>(m + 8 * j);
  double best = -INFINITY;
  // Four rows, or eight in two chains of MFMAs. Each chain is one block of code with the reads of its results: a
  // branch inside it (to leave the second out) led to reads without the wait that they need.
  auto rows = [&](int r0, auto groups_tag) __attribute__((always_inline)) {
    constexpr int kGroups = decltype(groups_tag)::value;
    u32x4 x[kGroups][kRun / 8];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint16_t* src = q + min(r0 + 4 * g + (lane & 3), s.group - 1) * q_sh + k * kRun;
#pragma unroll
      for (int j = 0; j < kRun / 8; ++j) x[g][j] = *reinterpret_cast<const u32x4*>(src + 8 * j);
    }
    double acc[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) acc[g] = 0.;
#pragma unroll
    for (int j = 0; j < kRun / 8; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double b = static_cast<double>(bf16_bits_to_f32(static_cast<uint16_t>(w[j][i / 2] >> (16 * (i & 1)))));
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const uint16_t a = static_cast<uint16_t>(x[g][j][i / 2] >> (16 * (i & 1)));
          acc[g] = __builtin_amdgcn_mfma_f64_4x4x4f64(
              static_cast<double>(kF16 ? f16_bits_to_f32(a) : bf16_bits_to_f32(a)), b, acc[g], 0, 0, 0);
        }
      }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) best = fmax(best, isnan(acc[g]) ? INFINITY : acc[g]);
  };
  for (int r0 = 0; r0 < s.group; r0 += 8) {
    if (r0 + 4 < s.group)
      rows(r0, std::integral_constant<int, 2>{});
    else
      rows(r0, std::integral_constant<int, 1>{});
  }
  best = fmax(best, __shfl_xor(best, 16));
  best = fmax(best, __shfl_xor(best, 32));
  return !there ? kAlways - 1 : at < s.first || at >= have - s.last ? kAlways : key_of(best);
}

template <int kD, bool kF16>
__global__ void __launch_bounds__(kThreads) page_scores_kernel(KvCache c, Select s, int blocks) {
  const int unit = blockIdx.x / blocks;
  const int u = unit % c.kv_heads, i = unit / c.kv_heads % s.tokens, b = unit / c.kv_heads / s.tokens;
  const Sight see = sight_of(c, s, b, i);
  const int tile = (blockIdx.x % blocks * kWaves + static_cast<int>(threadIdx.x >> 6)) * 16;
  if (tile >= see.have || see.have <= s.count) return;
  const uint16_t* q = s.q + b * s.q_sb + i * s.q_st + static_cast<int64_t>(u) * s.group * s.q_sh;
  const unsigned long long key = tile_keys<kD, kF16>(c, s, s.table + b * s.t_st, u, tile, see.have, q, s.q_sh);
  const int lane = threadIdx.x & 63;
  if (lane < 16 && tile + lane < see.have) s.keys[static_cast<int64_t>(unit) * s.width + tile + lane] = key;
}

__device__ __forceinline__ double value_of(unsigned long long key) {
  return __longlong_as_double(static_cast<long long>(key ^ (key >> 63 ? 1ull << 63 : ~0ull)));
}

// The `count` largest of n > count keys, of equal ones those in front. Few: a key per thread and its rank
// among all, which lie in LDS with zeros (less than any key) up to a multiple of 8. (Inlined, as the next one: as
// functions that kernels call they took 21.4 us instead of 20.4 for 128 of 8192 pages, scores included.)
__device__ __forceinline__ void take_by_rank(const unsigned long long* keys, int n, int count, const int* row, int* out) {
  __shared__ int s_sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = wave * 64;         // of the wave's keys
  int rank = count, page = 0;          // a wave without keys takes none
  if (first < n) {
    const int at = min(tid, n - 1);
    page = row[at];
    // in front of the wave's own keys an equal one counts as larger, behind them it does not
    const unsigned long long mine = keys[at];
    rank = 0;
    auto larger = [&](int j0, int j1, auto bound) __attribute__((always_inline)) {   // j0, j1 multiples of 8
      for (int j = j0; j < j1; j += 8) {
        unsigned long long k[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = keys[j + i];
#pragma unroll
        for (int i = 0; i < 8; ++i) rank += k[i] > bound(j + i);
      }
    };
    const int end = (n + 7) / 8 * 8;
    larger(0, first, [&](int) { return mine - 1; });
    larger(first, min(first + 64, end), [&](int j) { return j < tid ? mine - 1 : mine; });
    larger(first + 64, end, [&](int) { return mine; });
  }
  const bool taken = tid < n && rank < count;
  const unsigned long long all = __ballot(taken);
  if (lane == 0) s_sums[wave] = __popcll(all);
  __syncthreads();
  int before = __popcll(all & ((1ull << lane) - 1));
#pragma unroll
  for (int w = 0; w < kAloneThreads / 64; ++w) before += w < wave ? s_sums[w] : 0;
  if (taken) out[before] = page;
}

// Many. Thread t holds the keys t, t + threads, .. in registers, up to kRun of them, or, kRun = 0, reads
// them again for every step. With registers the scores go into as many bins as there are threads,
// evenly between the least and the largest finite one: the bin that the last taken one lies in has few
// others in it, and those are ranked. Where it has many (scores that are alike but for a few far off), and
// without registers, the least key that is taken is found by bisection, first between values, then
// between bit patterns. 128 of 8192 pages, 8 units: 10 us, by bisection 17.
constexpr int kMostRuns = 64, kMostWaves = kTakeThreads / 64;
constexpr int kMostInBin = 256;

template <int kRun>
__device__ __forceinline__ void take_many(const unsigned long long* keys, int n, int count, const int* row, int* out) {
  __shared__ int s_counts[3], s_before[(kRun > 0 ? kRun : kMostRuns) * kMostWaves];
  __shared__ unsigned long long s_low[kMostWaves], s_high[kMostWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int run = (n + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
  unsigned long long held[kRun > 0 ? kRun : 1];
  int ids[kRun > 0 ? kRun : 1];
  if constexpr (kRun > 0) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int j = min(tid + i * static_cast<int>(blockDim.x), n - 1);
      held[i] = keys[j];
      ids[i] = row[j];
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (tid + i * static_cast<int>(blockDim.x) >= n) held[i] = 0;   // less than any key
  }
  // f(key, whether it is one, page, turn) of every key of the thread; all lanes take part in every call
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (kRun > 0) {
#pragma unroll
      for (int i = 0; i < kRun; ++i) f(held[i], tid + i * static_cast<int>(blockDim.x) < n, ids[i], i);
    } else {
      for (int i = 0; i < run; ++i) {
        const int j = tid + i * static_cast<int>(blockDim.x);
        f(j < n ? keys[min(j, n - 1)] : 0ull, j < n, row[min(j, n - 1)], i);
      }
    }
  };
  // Turns the counts of s_before[turn][wave] into how many there are in front of each.
  auto scan_counts = [&]() __attribute__((always_inline)) {
    __syncthreads();
    if (wave == 0) {
      const int all = (kRun > 0 ? kRun : run) * waves, each_lane = (all + 63) / 64;
      int mine = 0;
      for (int i = lane * each_lane; i < min((lane + 1) * each_lane, all); ++i) mine += s_before[i];
      int incl = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(incl, d);
        incl += lane >= d ? other : 0;
      }
      int at = incl - mine;
      for (int i = lane * each_lane; i < min((lane + 1) * each_lane, all); ++i) {
        const int x = s_before[i];
        s_before[i] = at;
        at += x;
      }
    }
    __syncthreads();
  };
  const unsigned long long in_front = (1ull << lane) - 1;
  // Writes the pages whose bits are set, in order.
  auto write_taken = [&](unsigned long long taken) __attribute__((always_inline)) {
    __syncthreads();
    each([&](unsigned long long, bool, int, int i) {
      const int some = __popcll(__ballot(taken >> i & 1));
      if (lane == 0) s_before[i * waves + wave] = some;
    });
    scan_counts();
    each([&](unsigned long long, bool, int page, int i) {
      const bool mine = taken >> i & 1;
      const int at = s_before[i * waves + wave] + __popcll(__ballot(mine) & in_front);
      if (mine) out[at] = page;
    });
  };

  if constexpr (kRun > 0) {
    __shared__ int s_bins[kTakeThreads], s_sums[kMostWaves], s_bin[3];
    __shared__ float s_least[kMostWaves], s_most[kMostWaves];
    __shared__ unsigned long long s_list[kMostInBin];
    __shared__ int s_index[kMostInBin];
    __shared__ unsigned int s_taken[kRun * kTakeThreads / 32];
    const int threads = blockDim.x;
    // a key's score to fp32, which keeps the order; +inf for what always goes first
    float x[kRun], least = INFINITY, most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      x[i] = held[i] >= kAlways - 1 ? INFINITY : static_cast<float>(value_of(held[i]));
      const bool counts = held[i] != 0 && fabsf(x[i]) < INFINITY;
      least = fminf(least, counts ? x[i] : INFINITY);
      most = fmaxf(most, counts ? x[i] : -INFINITY);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      least = fminf(least, __shfl_xor(least, d));
      most = fmaxf(most, __shfl_xor(most, d));
    }
    if (lane == 0) {
      s_least[wave] = least;
      s_most[wave] = most;
    }
    s_bins[tid] = 0;
    for (int j = tid; j < kRun * kTakeThreads / 32; j += threads) s_taken[j] = 0;
    if (tid == 0) s_bin[2] = 0;
    __syncthreads();
    for (int w = 0; w < waves; ++w) {
      least = fminf(least, s_least[w]);
      most = fmaxf(most, s_most[w]);
    }
    const float per_bin = static_cast<float>(threads - 2) / (most - least);
    if (per_bin > 0.f && per_bin < INFINITY) {          // the same for all threads
      int bin[kRun];
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        bin[i] = x[i] == INFINITY ? threads - 1
                                  : static_cast<int>(fminf(fmaxf((x[i] - least) * per_bin, 0.f), threads - 2.f));
        if (held[i] != 0) atomicAdd(&s_bins[bin[i]], 1);
      }
      __syncthreads();
      const int mine = s_bins[threads - 1 - tid];       // from the last bin down
      int incl = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(incl, d);
        incl += lane >= d ? other : 0;
      }
      if (lane == 63) s_sums[wave] = incl;
      __syncthreads();
      int before = incl - mine;
      for (int w = 0; w < wave; ++w) before += s_sums[w];
      if (before < count && before + mine >= count) {
        s_bin[0] = threads - 1 - tid;
        s_bin[1] = count - before;
      }
      __syncthreads();
      const int last = s_bin[0], need = s_bin[1], in_bin = s_bins[last];
      if (in_bin == need || in_bin <= kMostInBin) {
        if (in_bin > need) {
#pragma unroll
          for (int i = 0; i < kRun; ++i)
            if (held[i] != 0 && bin[i] == last) {
              const int at = atomicAdd(&s_bin[2], 1);
              s_list[at] = held[i];
              s_index[at] = tid + i * threads;
            }
          __syncthreads();
          if (tid < in_bin) {
            const unsigned long long k = s_list[tid];
            const int index = s_index[tid];
            int rank = 0;
            for (int j = 0; j < in_bin; ++j) rank += s_list[j] > k || (s_list[j] == k && s_index[j] < index);
            if (rank < need) atomicOr(&s_taken[index >> 5], 1u << (index & 31));
          }
          __syncthreads();
        }
        unsigned long long taken = 0;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          const int index = tid + i * threads;
          const bool one = held[i] != 0 && (bin[i] > last || (bin[i] == last && (in_bin == need ||
                                                              (s_taken[index >> 5] >> (index & 31) & 1))));
          taken |= static_cast<unsigned long long>(one) << i;
        }
        write_taken(taken);
        return;
      }
    }
  }

  if (tid < 3) s_counts[tid] = 0;
  __syncthreads();
  int turn = 0;
  // Keys that `what` says yes to, over the workgroup: a ballot each, one atomic a wave, one barrier. The
  // three counters go round: one is summed, the last call's may still be read, the next call's is cleared.
  auto count_of = [&](auto what) __attribute__((always_inline)) {
    int mine = 0;
    each([&](unsigned long long k, bool there, int, int) { mine += __popcll(__ballot(what(k, there))); });
    if (lane == 0) atomicAdd(&s_counts[turn], mine);
    const int last = turn;
    turn = turn == 2 ? 0 : turn + 1;
    if (tid == 0) s_counts[turn] = 0;   // the next call's: it was read in front of the last barrier
    __syncthreads();
    return s_counts[last];
  };
  auto at_least = [&](unsigned long long bound) __attribute__((always_inline)) {
    return count_of([&](unsigned long long k, bool) { return k >= bound; });
  };

  // ---- bounds: at least `count` keys are >= low, less are >= high ----
  unsigned long long low, high;
  int found;                                   // keys that are >= low
  const int special = at_least(kAlways - 1);   // always taken, or pages that are not there
  if (special >= count) {
    const int always = at_least(kAlways);      // at most first + last <= count
    low = always >= count ? kAlways : kAlways - 1;
    found = always >= count ? always : special;
  } else {
    unsigned long long least = ~0ull, most = 0;
    each([&](unsigned long long k, bool there, int, int) {
      least = there && k < least ? k : least;
      most = k < kAlways - 1 && k > most ? k : most;
    });
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const unsigned long long a = __shfl_xor(least, d), b = __shfl_xor(most, d);
      least = a < least ? a : least;
      most = b > most ? b : most;
    }
    if (lane == 0) {
      s_low[wave] = least;
      s_high[wave] = most;
    }
    __syncthreads();
    for (int w = 0; w < waves; ++w) {
      least = s_low[w] < least ? s_low[w] : least;
      most = s_high[w] > most ? s_high[w] : most;
    }
    low = least;
    high = most + 1;
    found = n;
    for (int step = 0; found != count && high - low > 1; ++step) {
      unsigned long long middle = low + ((high - low) >> 1);
      if (step < 40) {
        const double m = 0.5 * value_of(low) + 0.5 * value_of(high - 1);
        const unsigned long long k = m == m ? key_of(m) : 0;
        if (k > low && k < high) middle = k;
      }
      const int some = at_least(middle);
      if (some >= count) {
        low = middle;
        found = some;
      } else {
        high = middle;
      }
    }
  }
  // ---- all above low, and of those that equal it (found is count: all of them) the first ones ----
  int need = n;
  if (found != count) {
    need = count - count_of([&](unsigned long long k, bool) { return k > low; });
    each([&](unsigned long long k, bool there, int, int i) {
      const int some = __popcll(__ballot(there && k == low));
      if (lane == 0) s_before[i * waves + wave] = some;
    });
    scan_counts();
  }
  unsigned long long taken = 0;      // a bit for each of the thread's keys
  each([&](unsigned long long k, bool there, int, int i) {
    const bool equal = there && k == low;
    const int before = need < n ? s_before[i * waves + wave] + __popcll(__ballot(equal) & in_front) : 0;
    taken |= static_cast<unsigned long long>(k > low || (equal && before < need)) << i;
  });
  write_taken(taken);
}

// What does not depend on scores: the tokens, and the pages where all are taken (true: nothing is left to do).
struct Unit {
  int b, i, u;
  const int* row;
  int* out;
  Sight see;
};
__device__ __forceinline__ bool take_all(const KvCache& c, const Select& s, Unit& at) {
  const int unit = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
  const int u = unit % c.kv_heads, i = unit / c.kv_heads % s.tokens, b = unit / c.kv_heads / s.tokens;
  at = {b, i, u, s.table + b * s.t_st, s.pages + static_cast<int64_t>(unit) * s.count, sight_of(c, s, b, i)};
  const Sight see = at.see;
  const int taken = min(max(see.have, 0), s.count);
  if (tid == 0) {
    if (see.have < 0) *c.faults = 1;
    if (u == 0)
      s.seen[unit / c.kv_heads] = see.have <= 0 ? see.tokens : see.tokens - ((see.have - taken) << c.log_page);
  }
  for (int j = taken + tid; j < s.count; j += threads) at.out[j] = -1;
  if (see.have > s.count) return false;
  for (int j = tid; j < taken; j += threads) at.out[j] = at.row[j];
  return true;
}

// Tables of up to so many pages keep their keys in LDS.
constexpr int kMostInLds = 8 * kAloneThreads;

template <int kD, bool kF16>
__global__ void __launch_bounds__(kAloneThreads) page_score_take_kernel(KvCache c, Select s) {
  extern __shared__ unsigned long long s_keys[];
  const int tid = threadIdx.x;
  Unit at;
  if (take_all(c, s, at)) return;
  const int have = at.see.have;
  const uint16_t* q = s.q + at.b * s.q_sb + at.i * s.q_st + static_cast<int64_t>(at.u) * s.group * s.q_sh;
  for (int tile = (tid >> 6) * 16; tile < have; tile += kAloneThreads / 64 * 16) {
    const unsigned long long key = tile_keys<kD, kF16>(c, s, at.row, at.u, tile, have, q, s.q_sh);
    if ((tid & 63) < 16) s_keys[tile + (tid & 15)] = tile + (tid & 15) < have ? key : 0;
  }
  __syncthreads();
  if (have <= kAloneThreads)
    take_by_rank(s_keys, have, s.count, at.row, at.out);
  else
    take_many<8>(s_keys, have, s.count, at.row, at.out);
}

__global__ void __launch_bounds__(kTakeThreads) page_take_kernel(KvCache c, Select s) {
  Unit at;
  if (take_all(c, s, at)) return;
  const unsigned long long* keys = s.keys + static_cast<int64_t>(blockIdx.x) * s.width;
  if (at.see.have <= 8 * kTakeThreads)
    take_many<8>(keys, at.see.have, s.count, at.row, at.out);
  else
    take_many<0>(keys, at.see.have, s.count, at.row, at.out);
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

constexpr int kMostPages = kMostRuns * kTakeThreads;
// Pages that one workgroup scores by itself where there are not many units
constexpr int kScoredAlone = 256;

bool scored_alone(int64_t units, int width) {
  return width <= kScoredAlone || (width <= kMostInLds && units >= 4ll * cu_count());
}

}  // namespace
}  // namespace vdn

using namespace vdn;

VDN_API int vdn_cache_means(const void* k_codes, const void* k_scales, int* faults, int pages, int kv_heads,
                            int page, int head_dim, const int* table, int64_t table_st, int batch, int width,
                            const int* starts, const int* lengths, void* means, void* stream) {
  const char* name = "vdn_cache_means";
  const KvCache c{static_cast<uint8_t*>(const_cast<void*>(k_codes)),
                  static_cast<uint8_t*>(const_cast<void*>(k_scales)), nullptr, nullptr, faults, pages, kv_heads,
                  page > 0 ? 31 - __builtin_clz(static_cast<unsigned>(page)) : 0};
  if (!cache_geometry_ok(c, page, head_dim) || batch < 0 || width <= 0)
    return set_error(kInvalidArgument,
                     "%s: bad geometry (page a power of two in 16..256, head_dim 64, 128 or 256)", name);
  if (batch == 0) return kOk;
  if (c.k == nullptr || c.ks == nullptr || faults == nullptr || table == nullptr || starts == nullptr ||
      lengths == nullptr || means == nullptr)
    return set_error(kInvalidArgument, "%s: null pointer", name);
  if (!aligned(c.k, 16) || !aligned(means, 16))
    return set_error(kInvalidArgument, "%s: codes and means need 16-byte alignment", name);
  const Spans s{table, starts, lengths, table_st, batch, width};
  // a wave per page and head, as many workgroups as run at once
  const int64_t most = (static_cast<int64_t>(batch) * width * kv_heads + kWaves - 1) / kWaves;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(most, 8ll * cu_count())));
  const auto st = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, c, s, static_cast<uint16_t*>(means));
  };
  head_dim == 64 ? launch(page_means_kernel<64>)
                 : head_dim == 128 ? launch(page_means_kernel<128>) : launch(page_means_kernel<256>);
  return check_launch(name);
}

VDN_API int vdn_cache_select_workspace(int batch, int tokens, int kv_heads, int width, int64_t* bytes) {
  if (bytes == nullptr || batch < 0 || tokens <= 0 || kv_heads <= 0 || width <= 0)
    return set_error(kInvalidArgument, "vdn_cache_select_workspace: invalid argument");
  const int64_t units = static_cast<int64_t>(batch) * tokens * kv_heads;
  *bytes = scored_alone(units, width) ? 0 : 8 * units * width;
  return kOk;
}

VDN_API int vdn_cache_select(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* means,
                             int* faults, int pages, int kv_heads, int page, int head_dim, const int* table,
                             int64_t table_st, int batch, int width, const int* lengths, int tokens, int group,
                             int dtype, int count, int first, int last, int* selected, int* seen, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const char* name = "vdn_cache_select";
  const KvCache c{nullptr, nullptr, nullptr, nullptr, faults, pages, kv_heads,
                  page > 0 ? 31 - __builtin_clz(static_cast<unsigned>(page)) : 0};
  if (!cache_geometry_ok(c, page, head_dim) || batch < 0 || width <= 0 || tokens <= 0 || group <= 0 ||
      width > kMostPages || (static_cast<int64_t>(width) << c.log_page) > (1ll << 31) - 1024)
    return set_error(kInvalidArgument, "%s: bad geometry (page a power of two in 16..256, head_dim 64, 128 or 256, "
                     "tables of at most %d pages)", name, kMostPages);
  if (dtype != 0 && dtype != 1) return set_error(kInvalidArgument, "%s: dtype must be 0 (bf16) or 1 (fp16)", name);
  if (first < 0 || last < 1 || count < 1 || first > count - last)
    return set_error(kInvalidArgument, "%s: first >= 0, last >= 1, and count at least both", name);
  if (batch == 0) return kOk;
  if (q == nullptr || means == nullptr || faults == nullptr || table == nullptr || lengths == nullptr ||
      selected == nullptr || seen == nullptr)
    return set_error(kInvalidArgument, "%s: null pointer", name);
  if (!aligned(q, 16) || !aligned(means, 16) || q_sb % 8 || q_st % 8 || q_sh % 8)
    return set_error(kInvalidArgument, "%s: queries and means need 16-byte alignment", name);
  const int64_t units = static_cast<int64_t>(batch) * tokens * kv_heads;
  const bool alone = scored_alone(units, width);
  const int64_t blocks = (static_cast<int64_t>(width) + 16 * kWaves - 1) / (16 * kWaves);
  // a grid has fewer than 2^32 threads: of kTakeThreads for a unit, of kThreads for 64 of its pages
  if (units * kTakeThreads >= (1ll << 32) || (!alone && units * blocks * kThreads >= (1ll << 32)))
    return set_error(kUnsupported, "%s: too many queries and pages", name);
  if (!alone && (workspace == nullptr || !aligned(workspace, 8) || workspace_bytes < 8 * units * width))
    return set_error(kInvalidArgument, "%s: workspace missing, unaligned or too small", name);
  const Select s{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(means), table, lengths, selected,
                 seen, alone ? nullptr : static_cast<unsigned long long*>(workspace), q_sb, q_st, q_sh, table_st,
                 batch, width, tokens, group, count, first, last};
  const auto st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(units));
  const auto launch = [&](auto scores, auto fused) {
    if (alone) {
      hipLaunchKernelGGL(fused, grid, dim3(kAloneThreads),
                         8u * static_cast<unsigned>((width + 15) / 16 * 16), st, c, s);
    } else {
      hipLaunchKernelGGL(scores, dim3(static_cast<unsigned>(units * blocks)), dim3(kThreads), 0, st, c, s,
                         static_cast<int>(blocks));
      hipLaunchKernelGGL(page_take_kernel, grid, dim3(kTakeThreads), 0, st, c, s);
    }
  };
#define VDN_SELECT(D, F16) launch(page_scores_kernel<D, F16>, page_score_take_kernel<D, F16>)
#define VDN_SELECT_D(F16) \
  head_dim == 64 ? VDN_SELECT(64, F16) : head_dim == 128 ? VDN_SELECT(128, F16) : VDN_SELECT(256, F16)
  if (dtype == 0)
    VDN_SELECT_D(false);
  else
    VDN_SELECT_D(true);
#undef VDN_SELECT_D
#undef VDN_SELECT
  return check_launch(name);
}

// Causal attention over packed prompts for gfx950 (bf16 or fp16; head_dim 64, 128, 256).
//
//   out[i, h] = sum_{j <= i} softmax_j(scale q[i, h] . k[j, u]) v[j, u],   u = h / G
//
// for the tokens i, j of one sequence; G query heads share the K/V head u. A sequence's n
// tokens and the G heads of u make n G rows, token major (row r: token r / G, head u G + r % G),
// and a workgroup takes a block of 32 kWaves of them: each K/V tile serves all G heads, and a
// block spans few tokens, so few of its tiles cross the diagonal.
//
// Per tile of kBN keys, as the frame-window kernel: Sᵀ = K Qᵀ on 32x32x16 MFMAs with Q in
// registers, online softmax in the exp2 domain (fp32 maximum and sum per row), and Oᵀ += Vᵀ Pᵀ,
// where Pᵀ is the Sᵀ accumulator itself and Vᵀ comes from the token-major V tile by transpose
// reads. P is rounded to 16 bits, the MFMA's operand, while its sum keeps fp32: errors of half a step
// each, which the sum over the keys averages (outputs within 2.1e-3 relative of 64 bits in bf16, where the
// output's own rounding makes 1.6e-3; 2.3e-4 and 2.0e-4 in fp16). Tiles stream global -> LDS,
// double-buffered. MFMA bounds long prompts, with the softmax beside it
// (63 and 49% of the time busy, the clock at 1.9 GHz by the power limit): 32768 tokens, 32 heads on 8
// x 128, 7.3 ms, 1200 TFLOP/s, 90% of a large library product. Short ones are bound by reading Q, writing
// O and the latency around the tiles: 24 prompts of 77 - 1200 tokens, 56 heads, 121 us.
//
// A nonfinite V value of a token that a row does not see must not reach that row, and 0 inf is
// NaN in an MFMA. Only tiles on the diagonal hold such tokens: there every wave looks its share
// of the V tile over as it lands, replaces nonfinite values by zeros and notes, per channel, the
// first token with a positive and with a negative one. What a row sees is a prefix, so the row
// holds that value exactly if the token is not behind its own: it is added after the last tile, when
// no wave changes the notes any more.
#include "attn_tiles.h"

#include <float.h>
#include <math.h>

#include <type_traits>

namespace vdn {
namespace {

// Maximum and sum over lanes l and l ^ 32 (the two halves of a row's keys), without LDS.
__device__ __forceinline__ float max_halves(float x) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

struct CausalIn {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token / head strides (elements)
};

// r / group for 0 <= r < 2^31, without a division: with s = ceil(log2 group) and mul = ceil(2^(31 + s) /
// group), r mul is r 2^(31 + s) / group and less than r <= 2^31 too much: the quotient stays.
struct GroupOf {
  uint32_t mul;
  int shift;   // 31 + s
  __device__ __forceinline__ int operator()(int r) const {
    return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(r)) * mul >> shift);
  }
};

struct CausalOut {
  uint16_t* out;
  float* lse;
  int64_t o_st, o_sh, l_st, l_sh;
};

// blocks: int32 [nblocks, 4] = (first token row, tokens n of the sequence, first row r0 of the
// block among the sequence's n G, unused), in the order of the launch.
// kWaves waves of 32 rows, tiles of kBN keys, kPerSimd waves on a SIMD (of one workgroup or of
// several); kSpread sends the next tile's loads out along Sᵀ instead of all at once.
template <int kD, int kWaves, int kBN, int kPerSimd, bool kSpread, bool kF16>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(kPerSimd, kPerSimd)))
causal_attn_kernel(CausalIn in, CausalOut to, const int* __restrict__ blocks, int nblocks,
                   int kv_heads, int together, int group, GroupOf token_of, float scale_log2) {
  constexpr int kKT = kBN / 32;           // 32-key score accumulators per tile
  constexpr int kDB = kD / 32;            // 32-channel output accumulators
  constexpr int kSteps = kD / 16;         // channel steps of Sᵀ
  constexpr int kChunks = kD / 8;         // 16-byte chunks per tile row
  constexpr int kSegRows = 64 / kChunks;  // rows per 1 KB DMA segment (one wave instruction)
  constexpr int kBM = 32 * kWaves;
  constexpr int kThreads = 64 * kWaves;
  constexpr int kLoaders = kSpread ? kWaves : kWaves / 2;  // the waves that load tiles (below)
  constexpr int kSegs = kBN / kSegRows / kLoaders;  // 1 KB segments per tensor per loading wave
  static_assert(kSegs * kLoaders * kSegRows == kBN, "segment mapping");
  static_assert(kBM <= 4 * kBN && kBN % 32 == 0, "the epilogue stages the block in the tile buffers");
  typedef Elem<kF16> E;
  typedef typename E::x8 x8;
  // one array per buffer: the compiler then tells a prefetch into one from reads of the other
  __shared__ __attribute__((aligned(1024))) uint16_t sK0[kBN * kD];
  __shared__ __attribute__((aligned(1024))) uint16_t sK1[kBN * kD];
  __shared__ __attribute__((aligned(1024))) uint16_t sV0[kBN * kD];
  __shared__ __attribute__((aligned(1024))) uint16_t sV1[kBN * kD];
  __shared__ int sPos[kD], sNeg[kD], sDirty;

  // With a multiple of 8 K/V heads each XCD keeps its own heads, so that a head's tiles are shared
  // in one L2; `together` of them go through the plan's blocks at a time. Otherwise consecutive ids
  // go round the XCDs.
  int u, blk;
  {
    const int pid = blockIdx.x;
    if (kv_heads % 8 == 0) {
      const int xcd = pid & 7, local = pid >> 3, turn = local / (together * nblocks);
      const int rest = local - turn * together * nblocks;
      blk = rest / together;
      u = xcd + 8 * (turn * together + rest - blk * together);
    } else {
      u = pid % kv_heads;
      blk = pid / kv_heads;
    }
  }
  const int64_t row0 = __builtin_amdgcn_readfirstlane(blocks[4 * blk]);
  const int n = __builtin_amdgcn_readfirstlane(blocks[4 * blk + 1]);
  const int r0 = __builtin_amdgcn_readfirstlane(blocks[4 * blk + 2]);
  const int rows = n * group;
  const int i_first = token_of(r0);                             // the block's tokens
  const int nkeys = token_of(min(r0 + kBM - 1, rows - 1)) + 1;   // keys that its last row sees
  const int ntiles = (nkeys + kBN - 1) / kBN;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, col = lane & 31;

  const int w0 = r0 + wave * 32;                 // the wave's rows
  const bool wave_live = w0 < rows;
  const int w_first = token_of(w0);
  const int w_last = token_of(min(w0 + 31, rows - 1));
  const int my_r = w0 + col;
  const bool live = my_r < rows;
  const int my_i = live ? token_of(my_r) : i_first;
  const int my_h = u * group + (live ? my_r - my_i * group : 0);

  // lane's share of a tile load: kSegs segments of kSegRows rows per tensor, at fixed byte
  // offsets from the tile's first row
  const int seg_row = lane / kChunks, phys = lane % kChunks;
  // Segments a multiple of 16 rows apart share the lane's swizzle: one offset per lane, the
  // segments' distance as the scalar one.
  constexpr int kApart = kLoaders * kSegRows;
  constexpr int kOffs = kApart % 16 == 0 ? 1 : kSegs;
  uint32_t koff[kOffs], voff[kOffs];
#pragma unroll
  for (int j = 0; j < kOffs; ++j) {
    const int row = (j * kLoaders + wave) * kSegRows + seg_row;
    koff[j] = static_cast<uint32_t>(row * in.k_st * 2 + 16 * (phys ^ swz_k<kD>(row)));
    voff[j] = static_cast<uint32_t>(row * in.v_st * 2 + 16 * (phys ^ swz_v<kD>(row)));
  }
  const char* k_head = reinterpret_cast<const char*>(in.k + row0 * in.k_st + u * in.k_sh);
  const char* v_head = reinterpret_cast<const char*>(in.v + row0 * in.v_st + u * in.v_sh);
  const uint32_t krow = static_cast<uint32_t>((wave * kSegRows + seg_row) * 2 * in.k_st);
  const uint32_t vrow = static_cast<uint32_t>((wave * kSegRows + seg_row) * 2 * in.v_st);
  struct Source {
    __amdgpu_buffer_rsrc_t k, v;
    int last;   // the tile's last row with a key; rows behind it repeat that
  };
  auto source = [&](int a) __attribute__((always_inline)) {
    return Source{tile_rsrc(k_head + static_cast<int64_t>(a) * in.k_st * 2),
                  tile_rsrc(v_head + static_cast<int64_t>(a) * in.v_st * 2), min(nkeys - 1 - a, kBN - 1)};
  };
  // segment j of 2 kSegs: K's, then V's
  auto issue_full = [&](const Source& src, int j, uint16_t* dk, uint16_t* dv) __attribute__((always_inline)) {
    const bool is_v = j >= kSegs;
    const int js = is_v ? j - kSegs : j, seg = js * kLoaders + wave;
    const uint32_t apart = kOffs > 1 ? 0 : static_cast<uint32_t>(js * kApart * (is_v ? in.v_st : in.k_st) * 2);
    load_to_lds16(is_v ? src.v : src.k, is_v ? voff[js % kOffs] : koff[js % kOffs], apart,
                  (is_v ? dv : dk) + seg * kSegRows * kD);
  };
  auto issue_tail = [&](const Source& src, int j, uint16_t* dk, uint16_t* dv) __attribute__((always_inline)) {
    const bool is_v = j >= kSegs;
    const int js = is_v ? j - kSegs : j, seg = js * kLoaders + wave, row = seg * kSegRows + seg_row;
    const uint32_t st = static_cast<uint32_t>(2 * (is_v ? in.v_st : in.k_st));
    const uint32_t at = min((is_v ? vrow : krow) + js * kApart * st, src.last * st);   // min(row, last) * st
    load_to_lds16(is_v ? src.v : src.k, at + 16 * (phys ^ (is_v ? swz_v<kD>(row) : swz_k<kD>(row))), 0,
                  (is_v ? dv : dk) + seg * kSegRows * kD);
  };
  auto issue_all = [&](int a, uint16_t* dk, uint16_t* dv) __attribute__((always_inline)) {
    const Source src = source(a);
    if (src.last == kBN - 1) {
#pragma unroll
      for (int j = 0; j < 2 * kSegs; ++j) issue_full(src, j, dk, dv);
    } else {
#pragma unroll
      for (int j = 0; j < 2 * kSegs; ++j) issue_tail(src, j, dk, dv);
    }
  };

  for (int d = tid; d < kD; d += kThreads) sPos[d] = sNeg[d] = 0x7fffffff;
  if (tid == 0) sDirty = 0;
  const bool loads = wave < kLoaders;
  if (loads) issue_all(0, sK0, sV0);

  // ---- Q fragments: row my_r, channels 16 ks + 8 g .. +8 ----
  x8 qf[kSteps];
  {
    const uint16_t* src = in.q + (row0 + my_i) * in.q_st + my_h * in.q_sh;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(src + 16 * ks + 8 * g);
      qf[ks] = __builtin_bit_cast(x8, w);
    }
  }

  f32x16 o[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  // m starts finite: a tile whose scores are all -inf then adds nothing instead of inf - inf
  float m = -FLT_MAX, l = 0.f;
  bool far = false;   // some row's m is beyond kFarScore
  // With one wave per SIMD half of the registers are accumulation registers, and O stays in them
  // if the rare branches that compute on it hand it back there; otherwise the compiler moves all
  // of O to the other half and back in every tile.
  auto keep = [&]() __attribute__((always_inline)) {
    if constexpr (kPerSimd == 1) {
#pragma unroll
      for (int db = 0; db < kDB; ++db) asm volatile("" : "+a"(o[db]));
    }
  };

  // transpose-read coordinates (16-lane group G = lane / 16)
  const int G = lane >> 4, L = lane & 15;
  const int tr_row = 4 * (G >> 1) + (L >> 2);
  const int tr_col = 16 * (G & 1) + 4 * (L & 3);

  // m is what the exponents are taken relative to (exp2 units): a row's running maximum less kAbove, which
  // may lag the true one by up to kLazy, so that most tiles need no rescale. Any m gives the same
  // weights; with kAbove those of fp16 reach up to 2^15, and one is rounded to within 2^-36 of the
  // largest instead of 2^-25 (32767 tokens of weight 2^-25 beside a heavy one would lose all of theirs).
  // bf16 has fp32's range.
  constexpr float kLazy = kF16 ? 4.f : 8.f, kAbove = kF16 ? 11.f : 0.f;
  auto process = [&](int t, auto buf_tag) __attribute__((always_inline)) {
    constexpr int kBuf = decltype(buf_tag)::value;
    const uint16_t* tk = kBuf == 0 ? sK0 : sK1;
    uint16_t* tv = kBuf == 0 ? sV0 : sV1;
    const int a = t * kBN;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of tile t is there
    const bool diagonal = a + kBN - 1 > i_first;      // some row does not see the whole tile
    if (diagonal && loads) {
      constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
#pragma unroll 1
      for (int j = 0; j < kSegs; ++j) {
        const int seg = j * kLoaders + wave;
        uint16_t* p = tv + seg * kSegRows * kD + lane * 8;
        u32x4 w = *reinterpret_cast<const u32x4*>(p);
        u16x2 mag = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        if (mag[0] < kInf && mag[1] < kInf) continue;
        const int row = seg * kSegRows + seg_row;
        const int ch = 8 * (phys ^ swz_v<kD>(row));
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const uint32_t b = p[i];
          if ((b & 0x7fffu) < kInf) continue;
          const bool nan = (b & 0x7fffu) > kInf;
          if (nan || b < 0x8000u) atomicMin(&sPos[ch + i], a + row);
          if (nan || b >= 0x8000u) atomicMin(&sNeg[ch + i], a + row);
          p[i] = 0;
        }
        sDirty = 1;
      }
    }
    __syncthreads();  // tile t is resident and every wave is done with the other buffer
    // The memory pipe takes 16 cycles for a segment, so a wave that issues many at once is held up
    // (about 70 cycles each). Two workgroups of 4 waves a CU: every wave loads its share, spread over
    // the channel steps of Sᵀ, in the shadow of its MFMAs (3% faster over 32768 tokens; V's along P V
    // instead came too late for the next tile). One workgroup of 8: waves 0 - 3, the older ones of
    // their SIMDs, come first through a tile and load for all behind their P V, where they would
    // wait for the others (3%; spread loads spill there). A tile with a tail, and a wave that sees
    // nothing of this tile, issue theirs here.
    uint16_t* ndk = kBuf == 0 ? sK1 : sK0;
    uint16_t* ndv = kBuf == 0 ? sV1 : sV0;
    const bool sees = wave_live && a <= w_last;
    const bool spread = kSpread && sees && nkeys - a >= 2 * kBN;
    const bool behind = !kSpread && sees;
    if (t + 1 < ntiles && !spread && !behind && loads) issue_all(a + kBN, ndk, ndv);
    if (!sees) return;
    const Source next = source(a + kBN);

    // ---- Sᵀ = K Qᵀ (kKT 32-key accumulators), the fragments of step ks + 1 read before the
    // MFMAs of step ks ----
    f32x16 s[kKT];
#pragma unroll
    for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[kt][v] = 0.f;
    x8 kf[2][kKT];
    auto kload = [&](int ks, x8 (&dst)[kKT]) __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt) {
        const int row = kt * 32 + col;
        const int chunk = (2 * ks + g) ^ swz_k<kD>(row);
        dst[kt] = *reinterpret_cast<const x8*>(tk + row * kD + chunk * 8);
      }
    };
    kload(0, kf[0]);
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      if (ks + 1 < kSteps) kload(ks + 1, kf[(ks + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt) s[kt] = E::mfma(kf[ks & 1][kt], qf[ks], s[kt]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kSpread) {
        constexpr int kEvery = kSteps / (2 * kSegs);
        static_assert(kEvery * 2 * kSegs == kSteps, "a segment every kEvery steps");
        if (spread && ks % kEvery == 0) issue_full(next, ks / kEvery, ndk, ndv);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // ---- online softmax ----
    if (a + kBN - 1 > w_first) {  // keys behind the row's token
      const int last = my_i - a - 4 * g;
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (kt * 32 + (v >> 2) * 8 + (v & 3) > last) s[kt][v] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[kt][v]);
    mx = max_halves(mx) * scale_log2;
    const bool grow = mx - m > kLazy + kAbove;
    if (__any(grow)) {
      const float m_new = grow ? below<kF16>(mx, kAbove) : m;
      const float corr = grow ? __builtin_amdgcn_exp2f(m - m_new) : 1.f;
      l *= corr;
      keep();
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= corr;
      keep();
      m = m_new;
      far = __any(fabsf(m) > kFarScore && m != -FLT_MAX);
    }
    float factor = scale_log2;
    if (__builtin_expect(far, 0)) {
      // m is the rounded product of a score and the scale: a score's own product has to be rounded like it.
      // (Following that costs up to 1%: two prompts of 4097 tokens, 16 heads on 1 x 256, 157.9 us against 156.1.)
#pragma unroll
      for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kt][v] *= scale_log2;
      factor = 1.f;
    }
    float rs = 0.f;
#pragma unroll
    for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][v], factor, -m));
        s[kt][v] = p;
        rs += p;
      }
    l += rs;   // of this lane's keys; the halves are joined at the end

    // ---- Oᵀ += Vᵀ Pᵀ, 16 keys per MFMA; the V fragments of MFMA i + kVA are read before
    // MFMA i ----
    constexpr int kItems = (kBN / 16) * kDB;
    constexpr int kVA = 2;
    x8 vf[kVA + 1];
    auto vload = [&](int i, x8& dst) __attribute__((always_inline)) {
      const int c = i / kDB, db = i % kDB;
      const int e = 32 * db + tr_col;
      const int lo_row = 16 * c + tr_row, hi_row = lo_row + 8;
      const typename E::x4 lo = E::read_tr(tv + lo_row * kD + ((e >> 3) ^ swz_v<kD>(lo_row)) * 8 + (e & 7));
      const typename E::x4 hi = E::read_tr(tv + hi_row * kD + ((e >> 3) ^ swz_v<kD>(hi_row)) * 8 + (e & 7));
      dst = x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
#pragma unroll
    for (int i = 0; i < kVA; ++i) vload(i, vf[i]);
    x8 pb;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (i + kVA < kItems) vload(i + kVA, vf[(i + kVA) % (kVA + 1)]);
      __builtin_amdgcn_sched_barrier(0x406);
      const int c = i / kDB, db = i % kDB;
      if (db == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pb[j] = static_cast<typename E::type>(s[c >> 1][(c & 1) * 8 + j]);
      }
      o[db] = E::mfma(vf[i % (kVA + 1)], pb, o[db]);
      __builtin_amdgcn_sched_barrier(0x406);
    }
    if (behind && loads && t + 1 < ntiles) issue_all(a + kBN, ndk, ndv);
  };
  __syncthreads();  // sPos, sNeg, sDirty
  for (int t = 0; t < ntiles; t += 2) {
    process(t, std::integral_constant<int, 0>{});
    if (t + 1 < ntiles) process(t + 1, std::integral_constant<int, 1>{});
  }
  keep();
  l = sum_halves(l);
  const float inv_l = l == 0.f ? NAN : 1.0f / l;   // l = 0 only if all scores are -inf: NaN, LSE -inf
  __syncthreads();                // the notes are final; the epilogue reuses the tile buffers
  if (sDirty != 0) {
    keep();
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int d = 32 * db + (v >> 2) * 8 + g * 4 + (v & 3);
        if (sPos[d] <= my_i) o[db][v] += INFINITY;
        if (sNeg[d] <= my_i) o[db][v] -= INFINITY;
      }
    keep();
  }

  // ---- epilogue: O / l through LDS to rows. Each wave stages its own 32 (no further barrier), four
  // channels a write; chunk c of row r lies at c ^ swz_k(r), so that the 32 rows of a write and the
  // rows of a read spread over the banks. ----
  const int first = wave * 32;
  uint16_t* sO = (first / kBN == 0 ? sK0 : first / kBN == 1 ? sK1 : first / kBN == 2 ? sV0 : sV1) +
                 first % kBN * kD;
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      typename E::x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // the rounded weights can take a mean of values next to fp16's largest one over it
        const float x = o[db][4 * j + i] * inv_l;
        y[i] = static_cast<typename E::type>(kF16 ? f16_in_range(x) : x);
      }
      *reinterpret_cast<typename E::x4*>(sO + col * kD + ((4 * db + j) ^ swz_k<kD>(col)) * 8 + 4 * g) = y;
    }
  if (to.lse != nullptr && live && g == 0)
    to.lse[(row0 + my_i) * to.l_st + my_h * to.l_sh] = (m + log2f(l)) * kLn2;
  const int64_t my_out = (row0 + my_i) * to.o_st + my_h * to.o_sh;
  const int out_lo = static_cast<int>(my_out), out_hi = static_cast<int>(my_out >> 32);
#pragma unroll
  for (int k = 0; k < 32; k += kSegRows) {
    const int r = k + seg_row;   // kChunks lanes a row
    const u32x4 row8 = *reinterpret_cast<const u32x4*>(sO + r * kD + (phys ^ swz_k<kD>(r)) * 8);
    const int64_t at = static_cast<int64_t>(__shfl(out_hi, r)) << 32 | static_cast<uint32_t>(__shfl(out_lo, r));
    if (w0 + r < rows) *reinterpret_cast<u32x4*>(to.out + at + phys * 8) = row8;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace vdn

using namespace vdn;

VDN_API int vdn_causal_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k,
                                 int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                                 int64_t v_sh, const int* blocks, int nblocks, int block_rows,
                                 int kv_heads, int group, int head_dim, int dtype, float scale,
                                 void* out, int64_t o_st, int64_t o_sh, float* lse, int64_t l_st,
                                 int64_t l_sh, void* stream) {
  const char* name = "vdn_causal_attention";
  if (nblocks < 0 || kv_heads <= 0 || group <= 0)
    return set_error(kInvalidArgument, "%s: bad geometry", name);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(kInvalidArgument, "%s: head_dim must be 64, 128 or 256", name);
  if (dtype != 0 && dtype != 1)
    return set_error(kInvalidArgument, "%s: dtype must be 0 (bf16) or 1 (fp16)", name);
  if (block_rows != 128 && (block_rows != 256 || head_dim != 128))
    return set_error(kInvalidArgument, "%s: block_rows must be 128, or 256 with head_dim 128", name);
  if (!(scale > 0.f) || !isfinite(scale)) return set_error(kInvalidArgument, "%s: bad scale", name);
  if (nblocks == 0) return kOk;
  if (q == nullptr || k == nullptr || v == nullptr || blocks == nullptr || out == nullptr)
    return set_error(kInvalidArgument, "%s: null pointer", name);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || q_st % 8 || q_sh % 8 ||
      k_st % 8 || k_sh % 8 || v_st % 8 || v_sh % 8 || o_st % 8 || o_sh % 8)
    return set_error(kInvalidArgument, "%s: rows need 16-byte alignment", name);
  // a lane's offset inside a tile of at most 128 keys is a 32-bit byte count
  if (k_st < 0 || v_st < 0 || k_st > (1 << 22) || v_st > (1 << 22))
    return set_error(kUnsupported, "%s: K/V token strides must be in [0, 2^22] elements", name);
  const int64_t total = static_cast<int64_t>(nblocks) * kv_heads;
  if (total * 512 >= (1ll << 32)) return set_error(kUnsupported, "%s: too many blocks", name);
  const CausalIn in{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k),
                    static_cast<const uint16_t*>(v), q_st, q_sh, k_st, k_sh, v_st, v_sh};
  const CausalOut to{static_cast<uint16_t*>(out), lse, o_st, o_sh, l_st, l_sh};
  // An XCD's heads all at once finish evenly, but their K/V no longer fits the L2: that pays as long
  // as all K/V fits the 256 MB cache behind it (a sequence's last block is counted in full). At once
  // against one after the other, tokens x heads of their own x 128, us: 2048 x 32 50, 59; 4096 x 32 138,
  // 181; 4096 x 56 241, 275; 8192 x 56 892, 987; 16384 x 32 (256 MB) 1932, 2014; 4 x 4096 x 56 1156,
  // 1016; 32768 x 32 8240, 7825. Many short prompts, which share little, do not follow the rule: 24 x 77 -
  // 1200 x 16 43, 42; 16 x 512 x 32 70, 65.
  const int64_t kv_bytes = static_cast<int64_t>(nblocks) * block_rows / group * head_dim * 4 * kv_heads;
  const int together = kv_heads % 8 == 0 && kv_bytes <= (256ll << 20) ? kv_heads / 8 : 1;
  const int ceil_log2 = group > 1 ? 32 - __builtin_clz(static_cast<unsigned>(group - 1)) : 0;
  const GroupOf token_of{static_cast<uint32_t>(((1ull << (31 + ceil_log2)) + group - 1) / group), 31 + ceil_log2};
  const auto launch = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(total)), dim3(threads), 0,
                       static_cast<hipStream_t>(stream), in, to, blocks, nblocks, kv_heads, together, group,
                       token_of, scale * kLog2e);
  };
  // 64 and 256 channels have one variant each. 64: three workgroups a CU (7% faster than two over 4 x
  // 4096 tokens of 32 heads, 18% over 64 prompts of 1 - 400; four spill). 256: Q and O alone take 192
  // registers, so one wave per SIMD with twice the registers (1.10 ms over 2 x 8192 tokens of 16
  // heads, 1040 TFLOP/s; two waves per SIMD spill and take 2.1).
#define VDN_CAUSAL(F16)                                                                          \
  head_dim == 64 ? launch(causal_attn_kernel<64, 4, 64, 3, true, F16>, 256)                      \
  : head_dim == 256 ? launch(causal_attn_kernel<256, 4, 64, 1, true, F16>, 256)                  \
  : block_rows == 256 ? launch(causal_attn_kernel<128, 8, 128, 2, false, F16>, 512)              \
                      : launch(causal_attn_kernel<128, 4, 64, 2, true, F16>, 256)
  if (dtype == 0)
    VDN_CAUSAL(false);
  else
    VDN_CAUSAL(true);
#undef VDN_CAUSAL
  return check_launch(name);
}

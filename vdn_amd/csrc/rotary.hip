// Rotation of queries and keys by their positions, with the RMSNorm of each head in front of it.
//
//   y = x rsqrt(sum(x^2) / D + eps) w                      (only with a weight)
//   (a, b) of pair j -> A (a cos t - b sin t, b cos t + a sin t),   t = position f_j,  j < R / 2
//
// Pair j is the channels (j, j + R/2) (half layout) or (2j, 2j + 1) (interleaved); channels from R on
// pass. All in fp32, rounded once at the end.
//
// The angle: f_j comes as a 64-bit fraction of a turn, so that position * f_j modulo 2^64 is the
// fraction of a turn without any error of the product, however far the position; its upper 32
// bits, less the nearest quarter turn, go to fp32 and to the Taylor polynomials of sin and cos on
// [-pi/4, pi/4] (x^9 and x^10: under 2^-28). A token's R/2 pairs are computed once for all its
// heads, and shared through LDS.
//
// A row's lane holds V = 8 (or 4) channels from V l and from R/2 + V l on (half layout) or 2 V from 2 V l on,
// so both channels of a pair are in one lane: no exchange but the norm's sum. Moving q and k once bounds
// it: 32768 tokens of 40 + 8 heads x 128, both norms, 805 MB in 139 - 147 us by card (5.8 - 5.5 TB/s; a large copy
// 5.1, a negation 6.3).
#include "common.h"

#include <math.h>

#include <algorithm>

namespace vdn {
namespace {

constexpr int kThreads = 256;
constexpr int kMostTokens = 16;   // of a workgroup

struct RotaryRows {
  const uint16_t* x;
  uint16_t* out;
  const void* w;                 // [D] or null
  int64_t st, sh, o_st, o_sh;    // token / head strides (elements)
};

struct RotaryArgs {
  RotaryRows q, k;
  const void* positions;
  const uint64_t* steps;   // [rot / 2] turns of one position, times 2^64
  int64_t tokens;
  int heads, all_heads;    // query heads; query and key heads
  int rot;
  int wide_positions, w_f32;
  int block_tokens;        // of a workgroup
  float amplitude, eps;
};

// cos and sin of the angle whose fraction of a turn is u / 2^32.
__device__ __forceinline__ void turn_cos_sin(uint32_t u, float* c, float* s) {
  const uint32_t quarter = (u + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int>(u - (quarter << 30))) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float x2 = x * x;
  const float sn = x + x * x2 * (-1.f / 6 + x2 * (1.f / 120 + x2 * (-1.f / 5040 + x2 * (1.f / 362880))));
  const float cs =
      1.f + x2 * (-0.5f + x2 * (1.f / 24 + x2 * (-1.f / 720 + x2 * (1.f / 40320 - x2 * (1.f / 3628800)))));
  const float a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
  *c = (quarter + 1) & 2 ? -a : a;   // quarters 1 and 2
  *s = quarter & 2 ? -b : b;
}

template <bool kF16>
__device__ __forceinline__ float widen(uint32_t w, int hi) {
  const uint16_t h = static_cast<uint16_t>(hi ? w >> 16 : w);
  return kF16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
}

// Streams past the caches: what is written is not read again here.
template <bool kF16, int kV>
__device__ __forceinline__ void store(const float* y, uint16_t* dst) {
  typedef unsigned int words __attribute__((ext_vector_type(kV / 2)));
  words r;
#pragma unroll
  for (int i = 0; i < kV / 2; ++i)
    r[i] = kF16 ? f32_to_f16_bits(y[2 * i]) | static_cast<uint32_t>(f32_to_f16_bits(y[2 * i + 1])) << 16
                : pack_bf16x2(y[2 * i], y[2 * i + 1]);
  __builtin_nontemporal_store(r, reinterpret_cast<words*>(dst));
}

template <int kD, bool kHalf, bool kF16, int kV>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a) {
  constexpr int kLanes = kD / (2 * kV);         // of a row
  typedef unsigned int words __attribute__((ext_vector_type(kV / 2)));
  constexpr int kRows = kThreads / kLanes;      // rows at a time
  __shared__ float s_cos[kMostTokens][kD / 2], s_sin[kMostTokens][kD / 2];
  __shared__ float s_w[2][kD];
  const int tid = threadIdx.x, l = tid % kLanes;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.block_tokens;
  const int n_tokens = static_cast<int>(min(static_cast<int64_t>(a.block_tokens), a.tokens - token0));
  const int rows = n_tokens * a.all_heads;
  const bool turned = 2 * kV * l < a.rot;
  const int c0 = kHalf && turned ? kV * l : 2 * kV * l;
  const int c1 = kHalf && turned ? a.rot / 2 + kV * l : 2 * kV * l + kV;

  struct Row {
    words lo, hi;
    int token, head;   // head: among queries and keys
  };
  auto load = [&](int r) __attribute__((always_inline)) {
    Row x;
    r = min(r, rows - 1);
    x.token = r / a.all_heads;
    x.head = r - x.token * a.all_heads;
    const bool is_k = x.head >= a.heads;
    const RotaryRows& io = is_k ? a.k : a.q;
    const uint16_t* p = io.x + (token0 + x.token) * io.st + (x.head - (is_k ? a.heads : 0)) * io.sh;
    x.lo = *reinterpret_cast<const words*>(p + c0);
    x.hi = *reinterpret_cast<const words*>(p + c1);
    return x;
  };
  int r = tid / kLanes;
  Row next = load(r);

  for (int i = tid; i < 2 * kD; i += kThreads) {
    const void* w = i < kD ? a.q.w : a.k.w;
    const int d = i % kD;
    if (w != nullptr)
      s_w[i / kD][d] = a.w_f32 ? static_cast<const float*>(w)[d]
                     : kF16 ? f16_bits_to_f32(static_cast<const uint16_t*>(w)[d])
                            : bf16_bits_to_f32(static_cast<const uint16_t*>(w)[d]);
  }
  const int pairs = a.rot / 2;
  for (int i = tid; i < n_tokens * (kD / 2); i += kThreads) {
    const int t = i / (kD / 2), j = i % (kD / 2);
    if (j >= pairs) continue;
    const int64_t at = token0 + t;
    const int64_t p = a.wide_positions ? static_cast<const int64_t*>(a.positions)[at]
                                       : static_cast<const int*>(a.positions)[at];
    float c, s;
    turn_cos_sin(static_cast<uint32_t>(static_cast<uint64_t>(p) * a.steps[j] >> 32), &c, &s);
    s_cos[t][j] = c * a.amplitude;
    s_sin[t][j] = s * a.amplitude;
  }
  __syncthreads();

  for (; r < rows; r += kRows) {
    const Row x = next;
    next = load(r + kRows);
    const bool is_k = x.head >= a.heads;
    float y[2 * kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      y[i] = widen<kF16>(x.lo[i / 2], i & 1);
      y[kV + i] = widen<kF16>(x.hi[i / 2], i & 1);
    }
    const RotaryRows& io = is_k ? a.k : a.q;
    if (io.w != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * kV; ++i) sum += y[i] * y[i];
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) sum += __shfl_xor(sum, d);
      const float scale = rsqrtf(sum * (1.f / kD) + a.eps);
#pragma unroll
      for (int j = 0; j < kV; j += 4) {
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(&s_w[is_k][c0 + j]);
        const f32x4 w1 = *reinterpret_cast<const f32x4*>(&s_w[is_k][c1 + j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[j + i] *= scale * w0[i];
          y[kV + j + i] *= scale * w1[i];
        }
      }
    }
    if (turned) {
#pragma unroll
      for (int j = 0; j < kV; j += 4) {
        const f32x4 c = *reinterpret_cast<const f32x4*>(&s_cos[x.token][kV * l + j]);
        const f32x4 s = *reinterpret_cast<const f32x4*>(&s_sin[x.token][kV * l + j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& p = kHalf ? y[j + i] : y[2 * (j + i)];
          float& q = kHalf ? y[kV + j + i] : y[2 * (j + i) + 1];
          const float u = p * c[i] - q * s[i], v = q * c[i] + p * s[i];
          p = u;
          q = v;
        }
      }
    }
    uint16_t* dst = io.out + (token0 + x.token) * io.o_st + (x.head - (is_k ? a.heads : 0)) * io.o_sh;
    store<kF16, kV>(y, dst + c0);
    store<kF16, kV>(y + kV, dst + c1);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace vdn

using namespace vdn;

VDN_API int vdn_rotary(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                       const void* q_w, const void* k_w, int w_f32, float eps, const void* positions,
                       int wide_positions, const void* steps, int rot, int interleaved, float amplitude,
                       int64_t tokens, int heads, int kv_heads, int head_dim, int dtype, void* qo,
                       int64_t qo_st, int64_t qo_sh, void* ko, int64_t ko_st, int64_t ko_sh, void* stream) {
  const char* name = "vdn_rotary";
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(kInvalidArgument, "%s: head_dim must be 64, 128 or 256", name);
  if (rot < 8 || rot > head_dim || rot % 8)
    return set_error(kInvalidArgument, "%s: rotated channels must be a multiple of 8 up to head_dim", name);
  if (tokens < 0 || heads <= 0 || kv_heads <= 0 || heads > 65536 || kv_heads > 65536)
    return set_error(kInvalidArgument, "%s: tokens >= 0, heads and kv_heads in 1..65536", name);
  if (dtype != 0 && dtype != 1) return set_error(kInvalidArgument, "%s: dtype must be 0 (bf16) or 1 (fp16)", name);
  if (!isfinite(amplitude) || !isfinite(eps) || eps < 0.f)
    return set_error(kInvalidArgument, "%s: bad amplitude or eps", name);
  if (tokens == 0) return kOk;
  if (q == nullptr || k == nullptr || positions == nullptr || steps == nullptr || qo == nullptr || ko == nullptr)
    return set_error(kInvalidArgument, "%s: null pointer", name);
  for (const int64_t s : {q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh})
    if (s % 4) return set_error(kInvalidArgument, "%s: rows need 8-byte alignment", name);
  for (const void* p : {q, k, static_cast<const void*>(qo), static_cast<const void*>(ko), steps})
    if (!aligned(p, 8)) return set_error(kInvalidArgument, "%s: rows need 8-byte alignment", name);
  if (!aligned(positions, wide_positions ? 8 : 4) || !aligned(q_w, w_f32 ? 4 : 2) || !aligned(k_w, w_f32 ? 4 : 2))
    return set_error(kInvalidArgument, "%s: positions and weights need their type's alignment", name);

  // 16-byte pieces where channels, strides and addresses allow them: 147 us against 172 with 8-byte ones
  // (32768 tokens, 40 + 8 heads x 128, both norms).
  bool wide = rot % 16 == 0;
  for (const int64_t s : {q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh}) wide &= s % 8 == 0;
  for (const void* p : {q, k, static_cast<const void*>(qo), static_cast<const void*>(ko)}) wide &= aligned(p, 16);
  // A workgroup has a token's heads, or those of several tokens where they are few: about three rows for
  // each place of a pass. Longer ones leave too few loads under way (4 tokens of 48 heads: 161 us against 147),
  // parts of a token's heads compute its angles again (200 us with one pass).
  const int all = heads + kv_heads, pass = kThreads / (head_dim / (wide ? 16 : 8));
  const int block_tokens = std::min(kMostTokens, std::max(1, 3 * pass / all));
  const int64_t blocks = (tokens + block_tokens - 1) / block_tokens;
  if (blocks > (1ll << 31) / kThreads) return set_error(kUnsupported, "%s: too many tokens", name);
  const RotaryArgs a{
      {static_cast<const uint16_t*>(q), static_cast<uint16_t*>(qo), q_w, q_st, q_sh, qo_st, qo_sh},
      {static_cast<const uint16_t*>(k), static_cast<uint16_t*>(ko), k_w, k_st, k_sh, ko_st, ko_sh},
      positions, static_cast<const uint64_t*>(steps), tokens, heads, all, rot, wide_positions, w_f32,
      block_tokens, amplitude, eps};
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
  };
#define VDN_ROT(D, V)                                                                                \
  interleaved ? (dtype ? launch(rotary_kernel<D, false, true, V>) : launch(rotary_kernel<D, false, false, V>)) \
              : (dtype ? launch(rotary_kernel<D, true, true, V>) : launch(rotary_kernel<D, true, false, V>))
#define VDN_ROT_V(D) wide ? (VDN_ROT(D, 8)) : (VDN_ROT(D, 4))
  if (head_dim == 64)
    VDN_ROT_V(64);
  else if (head_dim == 128)
    VDN_ROT_V(128);
  else
    VDN_ROT_V(256);
#undef VDN_ROT_V
#undef VDN_ROT
  return check_launch(name);
}

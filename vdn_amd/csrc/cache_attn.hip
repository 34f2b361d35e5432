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
  const int n_wg = sharers<false>(sp, total);
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
namespace units {

// Row blocks of 32 for more than 16 rows: every code is loaded and widened once for both halves.
// With 256 channels 32 rows spill (50.1 us against 50.4 in blocks of 16: 16 sequences of 4096
// tokens, 4 K/V heads, 32 rows), so those stay at 16.
int rows_of_block(int rows, int head_dim) { return rows > 16 && head_dim <= 128 ? 32 : 16; }

// As many workgroups as run at once, fewer if there are not so many quads at all.
int64_t workgroups_of(int64_t most_quads, int head_dim, int block) {
  const int64_t fit = static_cast<int64_t>(workgroups_per_cu(head_dim, block)) * cu_count();
  return std::max<int64_t>(1, std::min(fit, most_quads));
}

UnitPlan plan_units(int batch, int width, int log_page, int64_t rows, int kv_heads, int head_dim, int block) {
  UnitPlan p;
  p.block = block;
  p.row_blocks = static_cast<int>((rows + p.block - 1) / p.block);
  const int64_t unit_quads = ((static_cast<int64_t>(width) << log_page) + kQuad - 1) / kQuad;
  const int64_t all = static_cast<int64_t>(p.row_blocks) * kv_heads * batch;
  p.split = unit_quads > kWholeQuads;
  p.sp = Split{nullptr, static_cast<int>(workgroups_of(all * unit_quads, head_dim, p.block)),
               p.split ? kUnitCost : 0, 0, 0.f};
  p.slot_bytes = p.split ? 4ll * 2 * p.sp.workgroups * p.block * (head_dim + 4) : 0;
  return p;
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

// Whether the units of tables that a selection filled, most of them of the same length, are better left
// whole, a workgroup each: they are short, so that ragged ones do not cost more than the join does, and
// fill half of the places or more in each round. 64 queries of 384 tokens, 12 heads x 64: 12.6 us against 14.9;
// 32 of 2048 tokens, 40 heads on 8 x 128: 26.4, 30.9; 128: 107, 115; 64: 52.4, 53.9. (8192 tokens of
// 64 sequences of very different lengths would take 94 instead of 85.)
constexpr int kAlikeQuads = 8;
bool alike(int64_t units, int64_t places, int width, int log_page) {
  const int64_t quads = ((static_cast<int64_t>(width) << log_page) + kQuad - 1) / kQuad;
  const int64_t rounds = (units + places - 1) / places;
  return quads <= kAlikeQuads && 2 * units >= rounds * places;
}

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
  UnitPlan plan = plan_units(batch, width, c.log_page, rows, kv_heads, head_dim,
                             rows_of_block(static_cast<int>(std::min<int64_t>(rows, 32)), head_dim));
  const int64_t units = static_cast<int64_t>(plan.row_blocks) * kv_heads * batch;
  const bool one_each = table_sh != 0 && alike(units, plan.sp.workgroups, width, c.log_page);
  if (one_each) {
    plan.split = false;
    plan.sp.unit_cost = 0;
    plan.sp.workgroups = static_cast<int>(units);
  }
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
                       row_blocks, scale * kLog2e, static_cast<float*>(nullptr), NoFront{});
    if (!split) return;
    const dim3 grid(static_cast<unsigned>(join_rows));
    if (join_rows > 4 * cu_count())
      hipLaunchKernelGGL(join1, grid, dim3(64), 0, st, c, io, s, sp, row_blocks);
    else
      hipLaunchKernelGGL(join4, grid, dim3(256), 0, st, c, io, s, sp, row_blocks);
  };
  const Mode mode = one_each ? kOneEach : table_sh != 0 ? kShareHeads : kShare;
#define VDN_CACHE_AS(D, NR, F16, MODE) \
  launch(cache_attn_kernel<D, NR, F16, MODE, NoFront>, cache_join_kernel<D, NR, F16, 1>, cache_join_kernel<D, NR, F16, 4>)
#define VDN_CACHE(D, NR, F16)                                           \
  mode == kShare        ? VDN_CACHE_AS(D, NR, F16, kShare)              \
  : mode == kShareHeads ? VDN_CACHE_AS(D, NR, F16, kShareHeads)         \
                        : VDN_CACHE_AS(D, NR, F16, kOneEach)
#define VDN_CACHE_D(F16)                                                            \
  head_dim == 64 ? (block == 16 ? (VDN_CACHE(64, 1, F16)) : (VDN_CACHE(64, 2, F16)))    \
  : head_dim == 128 ? (block == 16 ? (VDN_CACHE(128, 1, F16)) : (VDN_CACHE(128, 2, F16))) \
                    : (VDN_CACHE(256, 1, F16))
  if (dtype == 0)
    VDN_CACHE_D(false);
  else
    VDN_CACHE_D(true);
#undef VDN_CACHE_D
#undef VDN_CACHE
#undef VDN_CACHE_AS
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

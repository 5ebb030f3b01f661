// Operators of libbwpp_hip around a transformer block: rotary positions, the
// residual join with its norms, and the cross entropy against a vocabulary,
// forward and gradient.  Argument checks, launch geometry and the choice of a
// kernel; the kernels are rotary.h, resnorm.h and xent.h.
#include "bwpp_hip.h"
#include "internal.h"

#include <algorithm>
#include <cmath>

#include "../kargs.h"

namespace {

enum LmKernel {
  LM_ROTARY_BF16,                      // [interleaved][chunk 8, 4, 1]
  LM_ROTARY_F32 = LM_ROTARY_BF16 + 6,  // [interleaved][chunk 4, 1]
  LM_RESNORM = LM_ROTARY_F32 + 4,      // [bf16][kResCfgs, any]
  LM_RESNORM_GRAD = LM_RESNORM + 14,   // [bf16][kResCfgs - 1, any]
  LM_RESNORM_FINISH = LM_RESNORM_GRAD + 14,  // [bf16]
  LM_XENT_JOIN = LM_RESNORM_FINISH + 2,
  LM_XENT_SUMS,
  LM_XENT_STATS_F32,
  LM_XENT_GRAD_F32,
  LM_XENT_TERMS,
  LM_XENT_ROUND,                         // fp32, bf16, bf16 with row-major W
  LM_XENT_CLEAR = LM_XENT_ROUND + 3,
  LM_XENT_COPY,                          // [bf16]
  LM_XENT_ZERO = LM_XENT_COPY + 2,       // [bf16]
  LM_XENT_STATS = LM_XENT_ZERO + 2,      // [trans_w][XentTile]
  LM_XENT_GRAD = LM_XENT_STATS + 14,
  LM_XENT_RAW = LM_XENT_GRAD + 14,
  LM_XENT_ROWS = LM_XENT_RAW + 14,
  LM_XENT_ROWS_RING,                     // XT_R32, XT_R64, XT_R128
  LM_XENT_ROW_SUMS = LM_XENT_ROWS_RING + 3,  // the same
  LM_TERMS_STATS = LM_XENT_ROW_SUMS + 3,                        // [trans_w][TermsTile]
  LM_TERMS_GRAD = LM_TERMS_STATS + 4,
  LM_TERMS_RAW = LM_TERMS_GRAD + 4,
  LM_TERMS_ROWS = LM_TERMS_RAW + 4,      // [TermsTile]
  LM_TERMS_RAW_T = LM_TERMS_ROWS + 2,    // [TermsTile]
  LM_COUNT = LM_TERMS_RAW_T + 2
};

// Rows in registers (resnorm.h): elements a thread and waves a row.
struct ResCfg {
  uint32_t elems, waves;
};
constexpr int kResNCfg = 6, kResGradNCfg = 6;
const ResCfg kResCfgs[kResNCfg] = {{8, 1}, {8, 2}, {8, 4}, {8, 8}, {8, 16}, {16, 16}};
const ResCfg kResGradCfgs[kResGradNCfg] = {{8, 1}, {16, 1}, {16, 2}, {16, 4}, {8, 8}, {16, 8}};
constexpr uint32_t kResAnyThreads = 512;

}  // namespace

const char *const bwpp_hip_lm_kernels[] = {
    "bwpp_rotary_bf16_half_8",      "bwpp_rotary_bf16_half_4",      "bwpp_rotary_bf16_half_1",
    "bwpp_rotary_bf16_inter_8",     "bwpp_rotary_bf16_inter_4",     "bwpp_rotary_bf16_inter_1",
    "bwpp_rotary_f32_half_4",       "bwpp_rotary_f32_half_1",       "bwpp_rotary_f32_inter_4",
    "bwpp_rotary_f32_inter_1",      "bwpp_resnorm_f32_n8_w1",       "bwpp_resnorm_f32_n8_w2",
    "bwpp_resnorm_f32_n8_w4",       "bwpp_resnorm_f32_n8_w8",       "bwpp_resnorm_f32_n8_w16",
    "bwpp_resnorm_f32_n16_w16",     "bwpp_resnorm_f32_any",         "bwpp_resnorm_bf16_n8_w1",
    "bwpp_resnorm_bf16_n8_w2",      "bwpp_resnorm_bf16_n8_w4",      "bwpp_resnorm_bf16_n8_w8",
    "bwpp_resnorm_bf16_n8_w16",     "bwpp_resnorm_bf16_n16_w16",    "bwpp_resnorm_bf16_any",
    "bwpp_resnorm_grad_f32_n8_w1", "bwpp_resnorm_grad_f32_n16_w1", "bwpp_resnorm_grad_f32_n16_w2",
    "bwpp_resnorm_grad_f32_n16_w4", "bwpp_resnorm_grad_f32_n8_w8", "bwpp_resnorm_grad_f32_n16_w8",
    "bwpp_resnorm_grad_f32_any",
    "bwpp_resnorm_grad_bf16_n8_w1", "bwpp_resnorm_grad_bf16_n16_w1", "bwpp_resnorm_grad_bf16_n16_w2",
    "bwpp_resnorm_grad_bf16_n16_w4", "bwpp_resnorm_grad_bf16_n8_w8", "bwpp_resnorm_grad_bf16_n16_w8",
    "bwpp_resnorm_grad_bf16_any",
    "bwpp_resnorm_finish_f32",      "bwpp_resnorm_finish_bf16",
    "bwpp_xent_join", "bwpp_xent_sums", "bwpp_xent_stats_f32", "bwpp_xent_grad_f32",
    "bwpp_xent_terms", "bwpp_xent_round_f32", "bwpp_xent_round_bf16", "bwpp_xent_round_bf16_dv",
    "bwpp_xent_clear", "bwpp_xent_copy_f32", "bwpp_xent_copy_bf16",
    "bwpp_xent_zero_f32", "bwpp_xent_zero_bf16",
    "bwpp_xent_stats_p_t00",
    "bwpp_xent_stats_r32_t00",
    "bwpp_xent_stats_r32_t00_u",
    "bwpp_xent_stats_r64_t00",
    "bwpp_xent_stats_r64_t00_u",
    "bwpp_xent_stats_r128_t00",
    "bwpp_xent_stats_r128_t00_u",
    "bwpp_xent_stats_p_t01",
    "bwpp_xent_stats_r32_t01",
    "bwpp_xent_stats_r32_t01_u",
    "bwpp_xent_stats_r64_t01",
    "bwpp_xent_stats_r64_t01_u",
    "bwpp_xent_stats_r128_t01",
    "bwpp_xent_stats_r128_t01_u",
    "bwpp_xent_grad_p_t00",
    "bwpp_xent_grad_r32_t00",
    "bwpp_xent_grad_r32_t00_u",
    "bwpp_xent_grad_r64_t00",
    "bwpp_xent_grad_r64_t00_u",
    "bwpp_xent_grad_r128_t00",
    "bwpp_xent_grad_r128_t00_u",
    "bwpp_xent_grad_p_t01",
    "bwpp_xent_grad_r32_t01",
    "bwpp_xent_grad_r32_t01_u",
    "bwpp_xent_grad_r64_t01",
    "bwpp_xent_grad_r64_t01_u",
    "bwpp_xent_grad_r128_t01",
    "bwpp_xent_grad_r128_t01_u",
    "bwpp_xent_sums_p_t00",
    "bwpp_xent_sums_r32_t00",
    "bwpp_xent_sums_r32_t00_u",
    "bwpp_xent_sums_r64_t00",
    "bwpp_xent_sums_r64_t00_u",
    "bwpp_xent_sums_r128_t00",
    "bwpp_xent_sums_r128_t00_u",
    "bwpp_xent_sums_p_t01",
    "bwpp_xent_sums_r32_t01",
    "bwpp_xent_sums_r32_t01_u",
    "bwpp_xent_sums_r64_t01",
    "bwpp_xent_sums_r64_t01_u",
    "bwpp_xent_sums_r128_t01",
    "bwpp_xent_sums_r128_t01_u",
    "bwpp_xent_rows_p_t10",
    "bwpp_xent_rows_r32_t10",
    "bwpp_xent_rows_r64_t10",
    "bwpp_xent_rows_r128_t10",
    "bwpp_xent_rowsums_r32_t10",
    "bwpp_xent_rowsums_r64_t10",
    "bwpp_xent_rowsums_r128_t10",
    "bwpp_xent_stats_sp_t00",
    "bwpp_xent_stats_sh_t00",
    "bwpp_xent_stats_sp_t01",
    "bwpp_xent_stats_sh_t01",
    "bwpp_xent_grad_sp_t00",
    "bwpp_xent_grad_sh_t00",
    "bwpp_xent_grad_sp_t01",
    "bwpp_xent_grad_sh_t01",
    "bwpp_xent_sums_sp_t00",
    "bwpp_xent_sums_sh_t00",
    "bwpp_xent_sums_sp_t01",
    "bwpp_xent_sums_sh_t01",
    "bwpp_xent_rows_sp_t10",
    "bwpp_xent_rows_sh_t10",
    "bwpp_xent_sums_sp_t10",
    "bwpp_xent_sums_sh_t10",
};
const int bwpp_hip_lm_kernel_count = (int)(sizeof(bwpp_hip_lm_kernels) / sizeof(bwpp_hip_lm_kernels[0]));
static_assert(sizeof(bwpp_hip_lm_kernels) / sizeof(bwpp_hip_lm_kernels[0]) == LM_COUNT, "kernel names");

// ------------------------------------- parameters, without their operands

namespace {

BwppHipFault invalid(const char *why) { return {BWPP_HIP_ERR_INVALID_ARG, why}; }
BwppHipFault unsupported(const char *why) { return {BWPP_HIP_ERR_UNSUPPORTED, why}; }
bool short_row(uint32_t ld, uint64_t cols) { return ld != 0 && ld < cols; }

}  // namespace

BwppHipFault bwpp_hip_check_rotary(const BwppRotaryParams &p) {
  if (p.dtype > BWPP_HIP_BF16) return invalid("unknown dtype");
  if (p.layout > BWPP_HIP_ROTARY_INTERLEAVED) return invalid("unknown layout");
  if (p.scaling > BWPP_HIP_ROTARY_SCALE_BY_PARTS) return invalid("unknown scaling");
  const uint32_t rot = p.rot_dim ? p.rot_dim : p.dim;
  if (rot % 2 || rot > p.dim) return invalid("rot_dim must be even and at most dim");
  if (!(p.base >= 0.0f) || !(p.factor >= 0.0f) || !std::isfinite(p.base) || !std::isfinite(p.factor) ||
      !std::isfinite(p.magnitude))
    return invalid("base and factor must be positive and finite, magnitude finite");
  if (p.scaling == BWPP_HIP_ROTARY_SCALE_BY_PARTS &&
      (p.context == 0 || !(p.high_turns > p.low_turns) || !std::isfinite(p.low_turns) || !std::isfinite(p.high_turns)))
    return invalid("scaling by parts needs a context and low_turns < high_turns");
  const uint64_t heads = (uint64_t)p.q_heads + p.k_heads;
  // (dim: a kernel's columns are 32-bit, and so is the end of a chunk that passes it)
  if (p.tokens && p.dim && (rot > 4096 || heads > (1u << 24) || p.tokens > (1u << 31) || p.dim > (1u << 31)))
    return unsupported("rot_dim above 4096, or dim, heads or tokens out of range");
  return {BWPP_HIP_OK, nullptr};
}

BwppHipFault bwpp_hip_check_residual_norm(const BwppResidualNormParams &p) {
  if (p.dtype > BWPP_HIP_BF16) return invalid("unknown dtype");
  if (short_row(p.ldx, p.cols) || short_row(p.ldo, p.cols) || short_row(p.ldy, p.cols) || short_row(p.ldg, p.cols))
    return invalid("row stride smaller than the row");
  if (!(p.eps >= 0.0f)) return invalid("eps must not be negative");
  if (p.cols >= (1u << 31)) return unsupported("2^31 columns or more");  // (32-bit columns are stepped past the row's end)
  return {BWPP_HIP_OK, nullptr};
}

BwppHipFault bwpp_hip_check_linear_xent(const BwppLinearXentParams &p) {
  if (p.dtype > BWPP_HIP_BF16) return invalid("unknown dtype");
  if (p.vocab == 0 || p.dim == 0) return invalid("empty vocabulary or dim");
  if (!std::isfinite(p.scale)) return invalid("scale must be finite");
  const uint64_t wcols = p.trans_w ? p.dim : p.vocab;
  if (short_row(p.ldx, p.dim) || short_row(p.ldw, wcols) || short_row(p.lddx, p.dim) || short_row(p.lddw, wcols))
    return invalid("row stride smaller than the row");
  if (p.rows >= (1u << 27) || p.vocab > 0x7fffffffu || p.dim > 0x7fffffffu)
    return unsupported("2^27 rows, or another size of 2^31, or more");
  if (p.dtype == BWPP_HIP_BF16 && (p.dim < 8 || (!p.trans_w && p.vocab < 8)))
    return unsupported("bf16 rows of fewer than 8 elements");
  return {BWPP_HIP_OK, nullptr};
}

namespace {

uint32_t cus_of(const BwppHip *h) {
  const int n = bwpp_hip_device_cus(h);
  return n > 0 ? (uint32_t)n : 256u;
}

// ---------------------------------------------------------------- rotary

// Rows of one operand of a rotary call: [batch][heads][tokens] rows of dim.
struct RowSet {
  const void *p;
  uint64_t ts, hs, bs;
  uint64_t batch, heads, tokens, dim;

  // A block of row stride ld that holds the set, where there is one: axes whose
  // strides are multiples of ld go along its rows, the others into a row.
  bool as_block(uint64_t ld, uint64_t &rows, uint64_t &cols) const {
    rows = 1;
    cols = dim;
    const uint64_t n[3] = {tokens, heads, batch}, st[3] = {ts, hs, bs};
    for (int i = 0; i < 3; ++i) {
      if (n[i] == 1) continue;
      if (st[i] % ld == 0) rows += (n[i] - 1) * (st[i] / ld);
      else cols += (n[i] - 1) * st[i];
    }
    return cols <= ld;
  }
  uint64_t span() const { return (batch - 1) * bs + (heads - 1) * hs + (tokens - 1) * ts + dim; }
};

// Whether two sets may share an element: not where they lie in blocks of one row
// stride, a token's, head's or batch's, that share none (q and k side by side in
// each token's row, or in each batch: heads before tokens); else by byte range.
bool meet(const RowSet &a, const RowSet &b, uint64_t es) {
  if (!a.p || !b.p) return false;
  for (const uint64_t ld : {a.tokens > 1 ? a.ts : 0, a.heads > 1 ? a.hs : 0, a.batch > 1 ? a.bs : 0}) {
    uint64_t ra, ca, rb, cb;
    if (ld && a.as_block(ld, ra, ca) && b.as_block(ld, rb, cb) &&
        !bwpp_hip_blocks_overlap(a.p, ra, ca, ld, b.p, rb, cb, ld, es))
      return false;
  }
  return bwpp_hip_blocks_overlap(a.p, 1, a.span(), 0, b.p, 1, b.span(), 0, es);
}
bool same_rows(const RowSet &a, const RowSet &b) {
  return a.p == b.p && (a.tokens == 1 || a.ts == b.ts) && (a.heads == 1 || a.hs == b.hs) &&
         (a.batch == 1 || a.bs == b.bs);
}
// Whether the rows of an output are disjoint: every stride passes what lies
// inside it, in some order of the three.
bool disjoint_rows(const RowSet &s) {
  struct Axis {
    uint64_t n, st;
  } ax[3] = {{s.tokens, s.ts}, {s.heads, s.hs}, {s.batch, s.bs}};
  std::sort(ax, ax + 3, [](const Axis &a, const Axis &b) { return a.st < b.st; });
  uint64_t inside = s.dim;
  for (const Axis &a : ax) {
    if (a.n == 1) continue;
    if (a.st < inside) return false;
    inside += (a.n - 1) * a.st;
  }
  return true;
}

BwppHipStatus rotary(BwppHip *h, const char *what, const void *q, const void *k, const int32_t *positions, void *qo,
                     void *ko, const BwppRotaryParams &p, bool grad) {
  auto bad = [&](const char *why) { return bwpp_hip_set_error(h, BWPP_HIP_ERR_INVALID_ARG, "%s: %s", what, why); };
  const BwppHipFault fault = bwpp_hip_check_rotary(p);
  if (fault.why) return bwpp_hip_set_error(h, fault.status, "%s: %s", what, fault.why);
  if (p.tokens == 0 || p.dim == 0 || (p.q_heads == 0 && p.k_heads == 0)) return bwpp_hip_enter(h);
  if ((p.q_heads && (!q || !qo)) || (p.k_heads && (!k || !ko))) return bad("NULL q, k or output");
  const uint32_t rot = p.rot_dim ? p.rot_dim : p.dim;
  const double base = p.base != 0.0f ? p.base : 10000.0, factor = p.factor != 0.0f ? p.factor : 1.0;
  const uint64_t B = p.batch ? p.batch : 1, T = p.tokens, d = p.dim, heads = (uint64_t)p.q_heads + p.k_heads;
  auto rows = [&](const void *ptr, uint32_t heads, uint32_t ld, uint64_t hs, uint64_t bs) {
    RowSet r = {heads ? ptr : nullptr, ld ? ld : d, 0, 0, B, heads ? heads : 1u, T, d};
    r.hs = hs ? hs : T * r.ts;
    r.bs = bs ? bs : r.heads * r.hs;
    return r;
  };
  // The gradient reads with the outputs' strides and writes with the inputs'.
  RowSet sq = rows(nullptr, p.q_heads, p.ldq, p.q_head_stride, p.q_batch_stride);
  RowSet sk = rows(nullptr, p.k_heads, p.ldk, p.k_head_stride, p.k_batch_stride);
  RowSet dq = rows(nullptr, p.q_heads, p.ldqo, p.qo_head_stride, p.qo_batch_stride);
  RowSet dk = rows(nullptr, p.k_heads, p.ldko, p.ko_head_stride, p.ko_batch_stride);
  if (grad) {
    std::swap(sq, dq);
    std::swap(sk, dk);
  }
  sq.p = p.q_heads ? q : nullptr;
  sk.p = p.k_heads ? k : nullptr;
  dq.p = p.q_heads ? qo : nullptr;
  dk.p = p.k_heads ? ko : nullptr;
  for (const RowSet *r : {&sq, &sk, &dq, &dk})
    if (r->p && T > 1 && r->ts < d) return bad("token stride smaller than the row");
  for (const RowSet *r : {&dq, &dk})
    if (r->p && !disjoint_rows(*r)) return bad("rows of an output overlap");
  const uint64_t es = p.dtype == BWPP_HIP_BF16 ? 2 : 4;
  if (positions) {
    const uint64_t bytes = ((B - 1) * p.pos_batch_stride + T) * 4;
    for (const RowSet *r : {&dq, &dk})
      if (r->p && bwpp_hip_blocks_overlap(r->p, 1, r->span() * es, 0, positions, 1, bytes, 0, 1))
        return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: an output overlaps the positions", what);
  }
  const bool q_in_place = sq.p && same_rows(sq, dq), k_in_place = sk.p && same_rows(sk, dk);
  if ((!q_in_place && meet(dq, sq, es)) || meet(dq, sk, es) || (!k_in_place && meet(dk, sk, es)) ||
      meet(dk, sq, es) || meet(dq, dk, es))
    return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: an output overlaps an input or the other output", what);
  const BwppHipStatus s = bwpp_hip_enter(h);
  if (s != BWPP_HIP_OK) return s;

  BwppRotaryArgs a = {};
  a.q = sq.p;
  a.k = sk.p;
  a.qo = const_cast<void *>(dq.p);
  a.ko = const_cast<void *>(dk.p);
  a.positions = positions;
  a.q_ts = sq.ts, a.q_hs = sq.hs, a.q_bs = sq.bs;
  a.k_ts = sk.ts, a.k_hs = sk.hs, a.k_bs = sk.bs;
  a.qo_ts = dq.ts, a.qo_hs = dq.hs, a.qo_bs = dq.bs;
  a.ko_ts = dk.ts, a.ko_hs = dk.hs, a.ko_bs = dk.bs;
  a.pos_bs = p.pos_batch_stride;
  a.log2_step = rot ? -2.0 / rot * std::log2(base) : 0.0;
  a.inv_factor = 1.0 / factor;
  a.turns = p.context * 0.15915494309189533577;  // 1 / (2 pi)
  a.low = p.low_turns;
  a.inv_range = p.scaling == BWPP_HIP_ROTARY_SCALE_BY_PARTS ? 1.0 / ((double)p.high_turns - (double)p.low_turns) : 0.0;
  a.cos_scale = p.magnitude != 0.0f ? p.magnitude : 1.0f;
  a.sin_scale = grad ? -a.cos_scale : a.cos_scale;
  a.pos0 = p.pos_offset;
  a.tokens = p.tokens;
  a.batch = (uint32_t)B;
  a.q_heads = p.q_heads;
  a.dim = p.dim;
  a.pairs = rot / 2;
  a.scaling = p.scaling;
  a.copy = rot < p.dim ? (sq.p && !q_in_place ? 1u : 0u) | (sk.p && !k_in_place ? 2u : 0u) : 0u;
  a.heads = (uint32_t)heads;
  const bool bf16 = p.dtype == BWPP_HIP_BF16, inter = p.layout == BWPP_HIP_ROTARY_INTERLEAVED;
  const uint32_t pick = bf16 ? (a.pairs % 8 == 0 ? 0u : a.pairs % 4 == 0 ? 1u : 2u) : (a.pairs % 4 == 0 ? 0u : 1u);
  const uint32_t chunk = bf16 ? (pick == 0 ? 8u : pick == 1 ? 4u : 1u) : (pick == 0 ? 4u : 1u);
  a.tail_chunks = a.copy ? (p.dim - rot + chunk - 1) / chunk : 0u;
  if (a.pairs == 0 && a.tail_chunks == 0) return BWPP_HIP_OK;
  // Tiles of tokens as wide as the angles' LDS allows while eight blocks a CU
  // remain; where there are few tokens the heads are split over blocks too.
  const uint64_t want = 8ull * cus_of(h);
  const uint32_t most = std::max(1u, 2048u / std::max(1u, a.pairs));
  a.tile = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(most, T), std::max<uint64_t>(1, B * T / want));
  a.hgroup = std::min(a.heads, 256u);
  const uint64_t blocks = B * ((T + a.tile - 1) / a.tile);
  while (a.hgroup > 8 && blocks * ((a.heads + a.hgroup - 1) / a.hgroup) * 2 <= want) a.hgroup = (a.hgroup + 1) / 2;
  const uint32_t groups = (a.heads + a.hgroup - 1) / a.hgroup;
  if (groups > 65535) return bwpp_hip_set_error(h, BWPP_HIP_ERR_UNSUPPORTED, "%s: too many heads", what);
  const int index = bf16 ? LM_ROTARY_BF16 + (inter ? 3 : 0) + (int)pick : LM_ROTARY_F32 + (inter ? 2 : 0) + (int)pick;
  return bwpp_hip_launch_lm(h, index, blocks, groups, 256, &a);
}

// --------------------------------------------------------- residual norm

// Checks and the arguments both directions share.
BwppHipStatus resnorm_prepare(BwppHip *h, const char *what, const BwppResidualNormParams &p, BwppResNormArgs &a) {
  const BwppHipFault fault = bwpp_hip_check_residual_norm(p);
  if (fault.why) return bwpp_hip_set_error(h, fault.status, "%s: %s", what, fault.why);
  a.rows = p.rows;
  a.cols = p.cols;
  a.ldx = p.ldx ? p.ldx : p.cols;
  a.ldo = p.ldo ? p.ldo : p.cols;
  a.ldy = p.ldy ? p.ldy : p.cols;
  a.ldg = p.ldg ? p.ldg : p.cols;
  a.post_norm = p.post_norm ? 1u : 0u;
  a.gate_rows = p.gate_rows;
  a.eps = p.eps;
  a.stream_scale = p.stream_scale != 0.0f ? p.stream_scale : 1.0f;
  a.branch_scale = p.branch_scale != 0.0f ? p.branch_scale : 1.0f;
  return BWPP_HIP_OK;
}

// Smallest layout whose threads hold a row, or -1: a block reads it again
// (as it does rows shorter than a chunk).
int res_cfg(uint32_t cols, const ResCfg *cfgs, int n) {
  if (cols < 8) return -1;
  for (int i = 0; i < n; ++i)
    if (64u * cfgs[i].elems * cfgs[i].waves >= cols) return i;
  return -1;
}

struct Block {
  const void *p;
  uint64_t rows, cols, ld;
};
bool meet(const Block &a, const Block &b, uint64_t es) {
  if (!a.p || !b.p || a.rows == 0 || b.rows == 0) return false;
  return bwpp_hip_blocks_overlap(a.p, a.rows, a.cols, a.ld, b.p, b.rows, b.cols, b.ld, es);
}

}  // namespace

extern "C" BwppHipStatus bwpp_hip_dispatch_rotary(BwppHip *h, const void *q, const void *k, const int32_t *positions,
                                                  void *qo, void *ko, BwppRotaryParams p) {
  return rotary(h, "rotary", q, k, positions, qo, ko, p, false);
}

extern "C" BwppHipStatus bwpp_hip_dispatch_rotary_grad(BwppHip *h, const void *dqo, const void *dko,
                                                       const int32_t *positions, void *dq, void *dk,
                                                       BwppRotaryParams p) {
  return rotary(h, "rotary_grad", dqo, dko, positions, dq, dk, p, true);
}

extern "C" BwppHipStatus bwpp_hip_dispatch_residual_norm(BwppHip *h, const void *x, const void *o,
                                                         const void *post_gamma, const void *gate,
                                                         const void *pre_gamma, void *r, void *y,
                                                         BwppResidualNormParams p) {
  if (p.rows && (!x || !o || !r)) return bwpp_hip_set_error(h, BWPP_HIP_ERR_INVALID_ARG, "residual_norm: NULL x, o or r");
  BwppResNormArgs a = {};
  BwppHipStatus s = resnorm_prepare(h, "residual_norm", p, a);
  if (s != BWPP_HIP_OK) return s;
  const uint64_t es = p.dtype == BWPP_HIP_BF16 ? 2 : 4, R = p.rows, C = p.cols;
  const uint64_t gates = p.gate_rows ? (R + p.gate_rows - 1) / p.gate_rows : 1;
  const Block bx = {x, R, C, a.ldx}, bo = {o, R, C, a.ldo}, br = {r, R, C, a.ldx}, by = {y, R, C, a.ldy};
  const Block small[3] = {{p.post_norm ? post_gamma : nullptr, 1, C, C}, {gate, gates, C, a.ldg}, {pre_gamma, 1, C, C}};
  bool alias = (x != r && meet(br, bx, es)) || meet(br, bo, es) || meet(br, by, es) || meet(by, bx, es) || meet(by, bo, es);
  for (const Block &b : small) alias = alias || meet(br, b, es) || meet(by, b, es);
  if (alias) return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "residual_norm: an output overlaps another operand");
  if ((s = bwpp_hip_enter(h)) != BWPP_HIP_OK || R == 0 || C == 0) return s;
  a.x = x;
  a.o = o;
  a.post = post_gamma;
  a.gate = gate;
  a.pre = pre_gamma;
  a.ro = r;
  a.y = y;
  const int c = res_cfg(p.cols, kResCfgs, kResNCfg), bf16 = p.dtype == BWPP_HIP_BF16;
  const uint32_t waves = c >= 0 ? kResCfgs[c].waves : 8u, rpb = waves == 1 ? 4u : 1u;
  // Blocks that keep the weights in registers over several rows.
  const uint64_t cap = (uint64_t)cus_of(h) * (waves >= 16 ? 2u : waves >= 8 ? 4u : 8u);
  const uint64_t blocks = std::min<uint64_t>((R + rpb - 1) / rpb, cap);
  return bwpp_hip_launch_lm(h, LM_RESNORM + bf16 * (kResNCfg + 1) + (c >= 0 ? c : kResNCfg), blocks, 1,
                            c < 0 ? kResAnyThreads : waves == 1 ? 256u : 64u * waves, &a);
}

extern "C" BwppHipStatus bwpp_hip_dispatch_residual_norm_grad(BwppHip *h, const void *o, const void *r,
                                                              const void *post_gamma, const void *gate,
                                                              const void *pre_gamma, const void *dr, const void *dy,
                                                              void *dx, void *dout, void *dpost_gamma, void *dgate,
                                                              void *dpre_gamma, BwppResidualNormParams p) {
  const char *what = "residual_norm_grad";
  auto bad = [&](const char *why) { return bwpp_hip_set_error(h, BWPP_HIP_ERR_INVALID_ARG, "%s: %s", what, why); };
  if (p.rows && (!o || !r || (!dr && !dy))) return bad("NULL o or r, or neither dr nor dy");
  if (p.rows && !dx && !dout && !dpost_gamma && !dgate && !dpre_gamma) return bad("no output");
  if (dpost_gamma && !p.post_norm) return bad("dpost_gamma without a post-norm");
  BwppResNormArgs a = {};
  BwppHipStatus s = resnorm_prepare(h, what, p, a);
  if (s != BWPP_HIP_OK) return s;
  const uint64_t es = p.dtype == BWPP_HIP_BF16 ? 2 : 4, R = p.rows, C = p.cols;
  if ((dpost_gamma || dgate || dpre_gamma) && (C + 63) / 64 * 1024 > 0xffffffffull)  // the sums' second launch
    return bwpp_hip_set_error(h, BWPP_HIP_ERR_UNSUPPORTED, "%s: weight or gate gradients of almost 2^28 columns or more", what);
  const uint64_t gates = p.gate_rows ? (R + p.gate_rows - 1) / p.gate_rows : 1;
  const Block in[7] = {{o, R, C, a.ldo}, {r, R, C, a.ldx}, {dr, R, C, a.ldx}, {dy, R, C, a.ldy},
                       {p.post_norm ? post_gamma : nullptr, 1, C, C}, {gate, gates, C, a.ldg}, {pre_gamma, 1, C, C}};
  const Block out[5] = {{dx, R, C, a.ldx}, {dout, R, C, a.ldo}, {dpost_gamma, 1, C, C}, {dgate, gates, C, a.ldg},
                        {dpre_gamma, 1, C, C}};
  for (int i = 0; i < 5; ++i) {
    for (int j = 0; j < 7; ++j)
      if (!(i == 0 && j == 2 && dx == dr) && meet(out[i], in[j], es))
        return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: an output overlaps an input", what);
    for (int j = 0; j < i; ++j)
      if (meet(out[i], out[j], es))
        return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: two outputs overlap", what);
  }
  if ((s = bwpp_hip_enter(h)) != BWPP_HIP_OK || C == 0) return s;
  if (R == 0 && p.gate_rows) dgate = nullptr;  // no gate rows
  if (R == 0 && !dgate && !dpost_gamma && !dpre_gamma) return BWPP_HIP_OK;
  a.o = o;
  a.r = r;
  a.post = post_gamma;
  a.gate = gate;
  a.pre = pre_gamma;
  a.dr = dr;
  a.dy = dy;
  a.dx = dx;
  a.dout = dout;
  a.dpost = dpost_gamma;
  a.dgate = dgate;
  a.dpre = dpre_gamma;
  const int c = res_cfg(p.cols, kResGradCfgs, kResGradNCfg), bf16 = p.dtype == BWPP_HIP_BF16;
  const uint32_t waves = c >= 0 ? kResGradCfgs[c].waves : 8u, rpb = waves == 1 ? 4u : 1u;
  // About `target` blocks, each of which leaves a partial row of every weight
  // gradient.  A group is what one row of dgate sums over; it is split over
  // blocks, or a worker takes whole groups.
  const uint64_t target = (uint64_t)cus_of(h) * (waves >= 8 ? 1u : waves >= 2 ? 8u / waves : bf16 ? 2u : 1u);
  const uint64_t group = dgate && p.gate_rows ? std::min<uint64_t>(p.gate_rows, std::max<uint64_t>(R, 1)) : std::max<uint64_t>(R, 1);
  const uint64_t ngroups = std::max<uint64_t>(1, (R + group - 1) / group);
  uint64_t split = 1, span, blocks;
  if (ngroups < target) {
    split = std::min<uint64_t>((target + ngroups - 1) / ngroups, std::max<uint64_t>(1, group / rpb));
    span = (group + split - 1) / split;
    split = (group + span - 1) / span;
  }
  if (split > 1) {
    a.workers = (uint32_t)(blocks = ngroups * split);
  } else {
    const uint64_t per = std::max<uint64_t>(1, (ngroups + target * rpb - 1) / (target * rpb));
    span = per * group;
    a.workers = (uint32_t)((ngroups + per - 1) / per);
    blocks = (a.workers + rpb - 1) / rpb;
  }
  if (span > 0xffffffffull) return bwpp_hip_set_error(h, BWPP_HIP_ERR_UNSUPPORTED, "%s: too many rows", what);
  a.group = (uint32_t)group;
  a.split = (uint32_t)split;
  a.span = (uint32_t)span;
  a.nparts = (uint32_t)blocks;
  const bool gate_part = dgate && (split > 1 || c < 0 || R == 0);
  const uint64_t nparts = (dpre_gamma ? 1 : 0) + (dpost_gamma ? 1 : 0) + (gate_part ? 1 : 0);
  if (nparts) {
    void *ws = nullptr;
    if ((s = bwpp_hip_take_workspace(h, nparts * blocks * C * sizeof(float), &ws)) != BWPP_HIP_OK) return s;
    float *f = static_cast<float *>(ws);
    if (dpre_gamma) a.part_pre = f, f += blocks * C;
    if (dpost_gamma) a.part_post = f, f += blocks * C;
    if (gate_part) a.part_gate = f;
  }
  s = bwpp_hip_launch_lm(h, LM_RESNORM_GRAD + bf16 * (kResGradNCfg + 1) + (c >= 0 ? c : kResGradNCfg),
                         blocks, 1, c < 0 ? kResAnyThreads : waves == 1 ? 256u : 64u * waves, &a);
  if (s != BWPP_HIP_OK || !nparts) return s;
  const bool gate_sum = gate_part && (split > 1 || R == 0);
  if (!gate_sum) a.part_gate = nullptr;
  if (!dpre_gamma && !dpost_gamma && !gate_sum) return BWPP_HIP_OK;
  return bwpp_hip_launch_lm(h, LM_RESNORM_FINISH + bf16, (C + 63) / 64, gate_sum ? 2u + (uint32_t)ngroups : 2u, 1024, &a);
}

// ------------------------------------------- cross entropy, vocabulary in pieces

namespace {

enum XentTile { XT_P, XT_R32, XT_R32U, XT_R64, XT_R64U, XT_R128, XT_R128U, XT_COUNT };
struct XentShape {
  uint32_t bm, bn, threads;
  double lat, inc, more;  // see xent_tile
};
const XentShape kXentShapes[XT_COUNT] = {
    {256, 256, 512, 0.0247, 0.0247, 3.0},  {32, 64, 128, 0.0039, 0.0032, 1.5},   {32, 64, 128, 0.0085, 0.0021, 1.5},
    {64, 64, 256, 0.0046, 0.0031, 0.6},    {64, 64, 256, 0.0088, 0.0040, 0.6},   {128, 128, 256, 0.0114, 0.0074, 1.4},
    {128, 128, 256, 0.0185, 0.0099, 1.4}};

bool on16(const void *p) { return ((uintptr_t)p & 15u) == 0; }
uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// The tile for a product A [M x K] op(B) [K x N] in the loops of gemm_bf16.h and
// gemm_bf16_k32.h: the DMA reads whole 16-byte chunks, the 256-wide tiles K in
// steps of 32; among those that can run, the one with the least modelled time.  n
// blocks on a CU take lat + (n - 1) inc us per K element and `more` each beyond the
// first (the constants that dispatch_matmul's choice was fitted with; 0.0247 for a
// round of 256-wide tiles, 8192^3 in 790 us), and no product runs faster than its
// operands arrive (5.6 TB/s; four fifths of it in the 128-byte pieces that 64
// columns take of row-major B: 42 x 704 x 69376 train 140 us on 64 x 64 tiles, 135
// on 128 x 128).  Sums: in planes of K ranges, as modelled; the 256-wide tiles' are
// chosen by the caller.
XentTile xent_tile(const BwppHip *h, const BwppGemmArgs &g, bool tb, bool sums, uint32_t *splits = nullptr) {
  const bool dma = on16(g.a) && on16(g.b) && g.lda % 8 == 0 && g.ldb % 8 == 0 && g.K % 8 == 0 && (tb || g.N % 8 == 0) &&
                   256ull * std::max(g.lda, g.ldb) < (1ull << 31);
  const uint64_t cus = cus_of(h);
  const double mem = ((double)g.M * g.K + (double)g.K * g.N) * 2.0 / 5.6e6;
  XentTile best = dma ? XT_R128 : XT_R128U;
  double best_us = 1e300;
  for (int t = 0; t < XT_COUNT; ++t) {
    const bool wide = t == XT_P, direct = wide || t == XT_R32 || t == XT_R64 || t == XT_R128;
    if (direct != dma || (wide && (sums || g.K % 32 != 0 || g.M <= 128))) continue;
    const XentShape &sh = kXentShapes[t];
    const uint64_t tiles = ((g.M + (uint64_t)sh.bm - 1) / sh.bm) * ((g.N + (uint64_t)sh.bn - 1) / sh.bn);
    // One range, or as many as fill 1 to 4 rounds of blocks.
    for (uint32_t rounds = 0; rounds <= (splits ? 4u : 0u); ++rounds) {
      const uint64_t fill = rounds ? std::min<uint64_t>(rounds * cus / tiles, std::min<uint64_t>(g.K / 256, 32)) : 1;
      if (rounds && fill < 2) continue;
      const uint32_t k = (uint32_t)fill;
      if (tiles * k * sh.threads > 0xffffffffull) continue;
      const double n = (double)((tiles * k + cus - 1) / cus);
      const double fetch = !tb && sh.bn == 64 ? mem * 1.25 : mem, planes = sums ? (double)k * g.M * g.N * 8.0 / 4e6 : 0.0;
      const double us = std::max(fetch, (n - 1.0) * sh.more + (double)g.K / k * (sh.lat + (n - 1.0) * sh.inc)) + planes;
      if (us < best_us * 0.999) {
        best_us = us;
        best = (XentTile)t;
        if (splits) *splits = k;
      }
    }
  }
  return best;
}

BwppHipStatus xent_product(BwppHip *h, int first, BwppXentArgs &a, bool tb, XentTile tile, uint32_t split) {
  const XentShape &sh = kXentShapes[tile];
  a.g.tiles_m = (uint32_t)((a.g.M + (uint64_t)sh.bm - 1) / sh.bm);
  a.g.tiles_n = (uint32_t)((a.g.N + (uint64_t)sh.bn - 1) / sh.bn);
  a.g.group_m = 8;
  a.g.kchunk = split > 1 ? (uint32_t)up((a.g.K + (uint64_t)split - 1) / split, 128) : a.g.K;
  split = (a.g.K + a.g.kchunk - 1) / a.g.kchunk;  // no empty range
  a.g.ksplit = split;
  const uint64_t tiles = (uint64_t)a.g.tiles_m * a.g.tiles_n;
  if (tiles > 0xffffffffull)
    return bwpp_hip_set_error(h, BWPP_HIP_ERR_UNSUPPORTED, "linear_xent: too many tiles");
  return bwpp_hip_launch_lm(h, first + (tb ? XT_COUNT : 0) + tile, tiles * split, 1, sh.threads, &a);
}

// Columns of a product on 256-wide tiles that smaller ones take instead: where
// the last round of tiles would leave half of the CUs idle or more, its tile
// columns (128 x 128 tiles, four for one, finish it in 0.4 to 0.7 of a round's
// time: 2048 tokens x 4096 x 50001, 6.1 rounds, 790 -> 739 us).
uint32_t xent_main_columns(const BwppHip *h, const BwppGemmArgs &g, XentTile tile) {
  const uint64_t tm = (g.M + 255ull) / 256, tn = (g.N + 255ull) / 256, cus = cus_of(h);
  if (tile != XT_P || tm * tn <= cus) return g.N;
  const uint64_t left = tm * tn % cus, columns = (left + tm - 1) / tm;
  return left == 0 || columns * tm * 2 > cus || columns >= tn ? g.N : (uint32_t)((tn - columns) * 256);
}

// The logits' product with the statistics' or the gradient's epilogue, in one
// launch or two.
uint32_t xent_tiles_n(const BwppHip *h, const BwppGemmArgs &g, XentTile tile) {
  const uint32_t n = xent_main_columns(h, g, tile);
  const uint32_t bn = kXentShapes[tile].bn;
  return (uint32_t)((n + (uint64_t)bn - 1) / bn) + (uint32_t)((g.N - n + 127ull) / 128);
}
BwppHipStatus xent_logits(BwppHip *h, int first, BwppXentArgs a, bool tb, XentTile tile) {
  const uint32_t n = xent_main_columns(h, a.g, tile), rest = a.g.N - n;
  a.g.N = n;
  const BwppHipStatus s = xent_product(h, first, a, tb, tile, 1);
  if (s != BWPP_HIP_OK || rest == 0) return s;
  a.part_base = a.g.tiles_n;
  a.g.b = static_cast<const uint16_t *>(a.g.b) + (tb ? (uint64_t)n * a.g.ldb : n);
  a.n_base += n;
  if (a.dl) a.dl += n;
  a.g.N = rest;
  return xent_product(h, first, a, tb, XT_R128, 1);
}

struct XentMatrices {
  uint64_t ldx, ldw, lddx, lddw, wrows, wcols;
};

BwppHipStatus xent_prepare(BwppHip *h, const char *what, const BwppLinearXentParams &p, XentMatrices &m) {
  const BwppHipFault fault = bwpp_hip_check_linear_xent(p);
  if (fault.why) return bwpp_hip_set_error(h, fault.status, "%s: %s", what, fault.why);
  m.wrows = p.trans_w ? p.vocab : p.dim;
  m.wcols = p.trans_w ? p.dim : p.vocab;
  m.ldx = p.ldx ? p.ldx : p.dim;
  m.ldw = p.ldw ? p.ldw : m.wcols;
  m.lddx = p.lddx ? p.lddx : p.dim;
  m.lddw = p.lddw ? p.lddw : m.wcols;
  return BWPP_HIP_OK;
}

// Columns of a piece: dz (bf16) or logits (fp32) of all rows in 256 MiB, which
// the Infinity Cache holds between the products, in whole tiles; at least 1024.
constexpr uint64_t kXentPiece = 256ull << 20;
uint32_t xent_piece(uint64_t rows, uint64_t vocab, uint64_t es) {
  uint64_t n = std::max<uint64_t>(kXentPiece / (std::max<uint64_t>(rows, 1) * es) / 256 * 256, 1024);
  if (n >= vocab) return (uint32_t)vocab;
  const uint64_t pieces = (vocab + n - 1) / n;
  n = up((vocab + pieces - 1) / pieces, 256);
  while (n < vocab && vocab % n != 0 && vocab % n < 8) n += 256;  // a last piece has a whole 16-byte chunk
  return (uint32_t)std::min(n, vocab);
}

// Few rows: a block for every 1024 columns of one.
uint32_t xent_columns(uint64_t rows, uint64_t cols) { return rows >= 1024 ? 1u : (uint32_t)std::min<uint64_t>((cols + 1023) / 1024, 256); }
uint32_t xent_grid(BwppHip *h, uint64_t rows) { return (uint32_t)std::min<uint64_t>(rows, 16ull * cus_of(h)); }

// Ends the hold on the workspace on every way out.
struct Hold {
  BwppHip *h;
  Hold(BwppHip *handle, size_t bytes) : h(handle) { bwpp_hip_hold_workspace(h, bytes); }
  ~Hold() { bwpp_hip_hold_workspace(h, 0); }
};
// Room behind the held part for the fp32 products' K splits.
constexpr size_t kXentSplitRoom = 64u << 20;

// z (unscaled) of the vocabulary's columns n0 .. n0 + n, fp32.
BwppHipStatus xent_logits_f32(BwppHip *h, const float *x, const float *w, float *z, uint32_t n0, uint32_t n,
                              const BwppLinearXentParams &p, const XentMatrices &m) {
  BwppMatmulParams g = {};
  g.M = p.rows;
  g.N = n;
  g.K = p.dim;
  g.lda = (uint32_t)m.ldx;
  g.ldb = (uint32_t)m.ldw;
  g.ldc = (uint32_t)up(n, 4);
  g.trans_b = p.trans_w ? 1u : 0u;
  return bwpp_hip_dispatch_matmul(h, x, w + (p.trans_w ? (uint64_t)n0 * m.ldw : n0), z, nullptr, g);
}

// ---- fp32 operands in bf16 terms (gemm_bf16_k32.h)

enum TermsTile { TT_P, TT_H };
struct TermsShape {
  uint32_t bm;
  double us;  // a round of tiles, per K element of one of the six products
};
constexpr TermsShape kTermsShapes[2] = {{256, 0.0252}, {128, 0.0163}};

// Terms of a matrix: four planes, or dz's three, of rows x cols up to multiples
// of 32.
struct Terms {
  uint16_t *p;
  uint64_t rows, cols;
  uint64_t plane() const { return up(rows * cols, 128); }
};
Terms terms_of(void *p, uint64_t rows, uint64_t cols) { return {static_cast<uint16_t *>(p), up(rows, 32), up(cols, 32)}; }
uint64_t terms_bytes(uint64_t rows, uint64_t cols, int planes) { return terms_of(nullptr, rows, cols).plane() * 2 * planes; }

// Modelled time of a product M x N x K in terms, and the tile that has it.
double terms_us(const BwppHip *h, uint64_t M, uint64_t N, uint64_t K, uint32_t split, TermsTile &tile) {
  double best = 1e300;
  for (int t = TT_P; t <= TT_H; ++t) {
    const uint64_t tiles = ((M + kTermsShapes[t].bm - 1) / kTermsShapes[t].bm) * ((N + 255) / 256) * split, cus = cus_of(h);
    const double us = 5.0 + (double)((tiles + cus - 1) / cus) * (3.0 + 6.0 * (double)((K + split - 1) / split) * kTermsShapes[t].us);
    if (us < best) best = us, tile = (TermsTile)t;
  }
  return std::max(best, (double)(M + N) * K * 12.0 / 3e6);  // six planes of each, from the Infinity Cache
}

// The same with K in ranges, summed in planes, where that is modelled faster by
// more than the planes cost.
double terms_split_us(const BwppHip *h, uint64_t M, uint64_t N, uint64_t K, uint32_t &split, TermsTile &tile, bool planes) {
  double best = terms_us(h, M, N, K, 1, tile) + (planes ? 5.0 + (double)M * N * 8.0 / 5e6 : 0.0);
  split = 1;
  for (uint32_t k = 2; k <= 8 && K / k >= 256; k *= 2) {
    TermsTile t;
    const double us = terms_us(h, M, N, K, k, t) + 5.0 + (double)k * M * N * 8.0 / 5e6;
    if (us < best) best = us, split = k, tile = t;
  }
  const uint64_t range = split > 1 ? up((K + split - 1) / split, 128) : K;  // as terms_product cuts it
  split = (uint32_t)((K + range - 1) / range);
  return best;
}

// Columns of a piece: its terms and dz's (gradient) in 256 MiB, and whole rounds of
// tiles of the logits, for few rows in up to 1 GiB.
uint32_t terms_piece(const BwppHip *h, const BwppLinearXentParams &p, bool grad) {
  const uint64_t bytes = 256 * (8 * up(p.dim, 32) + (grad ? 6 * up(p.rows, 32) : 0)), fits = kXentPiece / bytes;
  TermsTile tile;
  terms_us(h, p.rows, p.vocab, up(p.dim, 32), 1, tile);
  const uint64_t tm = (p.rows + kTermsShapes[tile].bm - 1) / kTermsShapes[tile].bm;
  const uint64_t round = std::min(std::max<uint64_t>(cus_of(h) / tm, 1), std::max<uint64_t>(4 * fits, 4));
  const uint64_t n = std::min<uint64_t>(std::max<uint64_t>(fits / round, 1) * round * 256, 1u << 22);
  return (uint32_t)std::min<uint64_t>(n, p.vocab);
}

// Whether a call's products go in terms: all of them as modelled, with the passes
// that make x's and W's (12 bytes an element), against fp32 matrix products at what
// they reach on such sizes (less where rows are no whole 16 bytes), logits through
// memory.  Loss and gradient, us, fp32 against terms: 1024 x 2048 x 8000 302 + 858
// against 248 + 599, 4096 x 2048 x 8000 1150 + 3295 against 683 + 1917; but 512 x 512
// x 4000 40 + 95 against 74 + 152, 256 x 2048 x 32000 280 + 803 against 464 + 1095.
bool xent_in_terms(const BwppHip *h, const BwppLinearXentParams &p, const XentMatrices &m, bool grad) {
  const uint64_t K = up(p.dim, 32), T = p.rows;
  if (T <= 128 || K > (1u << 22)) return false;
  const uint32_t piece = terms_piece(h, p, grad);
  const double D = p.dim, V = p.vocab, rate = m.ldx % 4 == 0 && m.ldw % 4 == 0 ? 105e6 : 80e6;
  const double fp32 = 2.0 * T * D * V / rate + 10.0;
  double us = ((double)T + V) * D * 12.0 / 5e6 + 8.0;
  const double old = T * V * 8.0 / 4.5e6 + (grad ? 3.0 : 1.0) * fp32;
  const uint64_t count[2] = {p.vocab / piece, p.vocab % piece ? 1u : 0u}, size[2] = {piece, p.vocab % piece};
  for (int i = 0; i < 2; ++i) {
    if (!count[i]) continue;
    TermsTile tile;
    uint32_t split;
    double one = 5.0 + terms_us(h, T, size[i], K, 1, tile);
    if (grad)
      one += terms_split_us(h, T, p.dim, up(size[i], 32), split, tile, true) +
             terms_split_us(h, p.dim, size[i], up(T, 32), split, tile, false);
    us += (double)count[i] * one;
  }
  return us < old;
}

BwppHipStatus make_terms(BwppHip *h, const float *src, uint64_t ld, uint64_t rows, uint64_t cols, const Terms &t,
                         const int32_t *targets, uint32_t vocab) {
  BwppXentRowArgs r = {};
  r.x = src;
  r.y = t.p;
  r.ldx = ld;
  r.ldy = t.cols;
  r.rows = (uint32_t)rows;
  r.cols = (uint32_t)cols;
  r.rows_up = (uint32_t)t.rows;
  r.plane = t.plane();
  r.target = targets;
  r.vocab = vocab;
  r.lanes = 4;
  while (r.lanes < 256 && r.lanes * 8 < t.cols) r.lanes *= 2;
  const uint64_t blocks = (t.rows + 256 / r.lanes - 1) / (256 / r.lanes);
  return bwpp_hip_launch_lm(h, LM_XENT_TERMS, std::min<uint64_t>(blocks, 32ull * cus_of(h)), 1, 256, &r);
}

// Six products as one.  Planes, smallest first: 3 = third, 2 = second, 1 = first
// where finite, 0 = first; of dz 2, 1, 0.
constexpr uint32_t kTermsA = 0x012213, kTermsAz = 0x001102, kTermsB = 0x021231, kTermsBz = 0x010120;
BwppHipStatus terms_product(BwppHip *h, int first, BwppXentArgs &a, bool tb, const Terms &A, const Terms &B, bool za, bool zb,
                            TermsTile tile, uint32_t split) {
  a.g.a = A.p;
  a.g.b = B.p;
  a.g.lda = (uint32_t)A.cols;
  a.g.ldb = (uint32_t)B.cols;
  a.terms.a_planes = za ? kTermsAz : kTermsA;
  a.terms.b_planes = zb ? kTermsBz : kTermsB;
  a.terms.a_stride = A.plane();
  a.terms.b_stride = B.plane();
  a.g.tiles_m = (uint32_t)((a.g.M + (uint64_t)kTermsShapes[tile].bm - 1) / kTermsShapes[tile].bm);
  a.g.tiles_n = (uint32_t)((a.g.N + 255ull) / 256);
  a.g.group_m = 8;
  a.g.kchunk = split > 1 ? (uint32_t)up((a.g.K + (uint64_t)split - 1) / split, 128) : a.g.K;
  a.g.ksplit = (a.g.K + a.g.kchunk - 1) / a.g.kchunk;
  const uint64_t tiles = (uint64_t)a.g.tiles_m * a.g.tiles_n * a.g.ksplit;
  if (tiles * 512 > 0xffffffffull) return bwpp_hip_set_error(h, BWPP_HIP_ERR_UNSUPPORTED, "linear_xent: too many tiles");
  return bwpp_hip_launch_lm(h, first + (tb ? 2 : 0) + tile, tiles, 1, 512, &a);
}

// One piece of the vocabulary: W's rows or columns n0 .. n0 + n in terms.
BwppHipStatus piece_terms(BwppHip *h, const float *w, const BwppLinearXentParams &p, const XentMatrices &m, uint32_t n0,
                          uint32_t n, Terms &wt, void *room) {
  wt = p.trans_w ? terms_of(room, n, p.dim) : terms_of(room, p.dim, n);
  return make_terms(h, w + (p.trans_w ? (uint64_t)n0 * m.ldw : n0), m.ldw, p.trans_w ? n : p.dim, p.trans_w ? p.dim : n, wt,
                    nullptr, 0);
}

BwppHipStatus terms_stats(BwppHip *h, const float *x, const float *w, const BwppLinearXentParams &p, const XentMatrices &m,
                          uint64_t front, BwppXentRowArgs &r, void *&ws) {
  const bool tw = p.trans_w != 0;
  const uint64_t T = p.rows, K = up(p.dim, 32);
  const uint32_t piece = terms_piece(h, p, false);
  const uint64_t npieces = (p.vocab + (uint64_t)piece - 1) / piece;
  // (a piece is a multiple of 256 columns, or the only one)
  r.nparts = (uint32_t)((p.vocab + 255ull) / 256);
  const uint64_t part_bytes = up((uint64_t)r.nparts * T * 8, 256), x_bytes = terms_bytes(T, p.dim, 4);
  const uint64_t w_bytes = terms_bytes(piece, p.dim, 4);
  BwppHipStatus s = bwpp_hip_take_workspace(h, front + part_bytes + x_bytes + w_bytes, &ws);
  if (s != BWPP_HIP_OK) return s;
  unsigned char *base = static_cast<unsigned char *>(ws) + front;
  r.zt = static_cast<float *>(ws);
  r.part = reinterpret_cast<float *>(base);
  const Terms xt = terms_of(base + part_bytes, T, p.dim);
  if ((s = make_terms(h, x, m.ldx, T, p.dim, xt, nullptr, 0)) != BWPP_HIP_OK) return s;
  for (uint64_t i = 0; i < npieces; ++i) {
    const uint32_t n0 = (uint32_t)(i * piece), n = std::min(piece, p.vocab - n0);
    Terms wt;
    if ((s = piece_terms(h, w, p, m, n0, n, wt, base + part_bytes + x_bytes)) != BWPP_HIP_OK) return s;
    BwppXentArgs a = {};
    a.g.M = p.rows;
    a.g.N = n;
    a.g.K = (uint32_t)K;
    a.target = r.target;
    a.vocab = p.vocab;
    a.scale = r.scale;
    a.n_base = n0;
    a.part_base = n0 / 256;
    a.zt = r.zt;
    a.part = r.part;
    TermsTile tile;
    terms_us(h, a.g.M, a.g.N, K, 1, tile);
    if ((s = terms_product(h, LM_TERMS_STATS, a, tw, xt, wt, false, false, tile, 1)) != BWPP_HIP_OK) return s;
  }
  return BWPP_HIP_OK;
}

BwppHipStatus terms_grad(BwppHip *h, const float *x, const float *w, float *dx, float *dw, const BwppLinearXentParams &p,
                         const XentMatrices &m, BwppXentRowArgs &r) {
  const bool tw = p.trans_w != 0;
  const uint64_t T = p.rows, D = p.dim, K = up(D, 32);
  const uint32_t piece = terms_piece(h, p, true);
  const uint64_t npieces = (p.vocab + (uint64_t)piece - 1) / piece;
  uint32_t split = 1, dw_split = 1;
  TermsTile dx_tile, dw_tile;
  terms_split_us(h, T, D, up(piece, 32), split, dx_tile, true);
  terms_split_us(h, tw ? piece : D, tw ? D : piece, up(T, 32), dw_split, dw_tile, false);
  const uint64_t x_bytes = terms_bytes(T, D, 4), w_bytes = terms_bytes(piece, D, 4), z_bytes = terms_bytes(T, piece, 3);
  const uint64_t sum_bytes = dx ? up(split * T * D * 4, 256) : 0, dw_bytes = dw && dw_split > 1 ? dw_split * piece * D * 4 : 0;
  void *ws = nullptr;
  BwppHipStatus s = bwpp_hip_take_workspace(h, x_bytes + w_bytes + z_bytes + sum_bytes + dw_bytes, &ws);
  if (s != BWPP_HIP_OK) return s;
  unsigned char *base = static_cast<unsigned char *>(ws);
  float *acc = reinterpret_cast<float *>(base + x_bytes + w_bytes + z_bytes);
  const Terms xt = terms_of(base, T, D);
  if ((s = make_terms(h, x, m.ldx, T, D, xt, r.target, p.vocab)) != BWPP_HIP_OK) return s;
  for (uint64_t i = 0; i < npieces; ++i) {
    const uint32_t n0 = (uint32_t)(i * piece), n = std::min(piece, p.vocab - n0);
    Terms wt;
    if ((s = piece_terms(h, w, p, m, n0, n, wt, base + x_bytes)) != BWPP_HIP_OK) return s;
    const Terms zt = terms_of(base + x_bytes + w_bytes, T, n);
    BwppXentArgs a = {};
    TermsTile tile;
    a.g.M = p.rows;
    a.g.N = n;
    a.g.K = (uint32_t)K;
    a.target = r.target;
    a.lse = r.lse_in;
    a.dloss = r.dloss;
    a.dloss_scalar = r.dloss_scalar;
    a.vocab = p.vocab;
    a.scale = r.scale;
    a.n_base = n0;
    a.dl = zt.p;
    a.ldl = (uint32_t)zt.cols;
    a.rows_up = (uint32_t)zt.rows;
    a.cols_up = (uint32_t)zt.cols;
    a.dl_stride = zt.plane();
    terms_us(h, T, n, K, 1, tile);
    if ((s = terms_product(h, LM_TERMS_GRAD, a, tw, xt, wt, false, false, tile, 1)) != BWPP_HIP_OK) return s;
    if (dx) {
      BwppXentArgs q = {};
      q.g.M = p.rows;
      q.g.N = p.dim;
      q.g.K = (uint32_t)zt.cols;
      q.raw = acc;
      q.accumulate = i > 0;
      // A last piece with fewer ranges leaves the others' sums as they are.
      if ((s = terms_product(h, LM_TERMS_RAW, q, !tw, zt, wt, true, false, dx_tile, split)) != BWPP_HIP_OK) return s;
    }
    if (dw) {
      BwppXentArgs q = {};
      q.g.M = tw ? n : p.dim;
      q.g.N = tw ? p.dim : n;
      q.g.K = (uint32_t)xt.rows;
      q.g.c = dw + (tw ? (uint64_t)n0 * m.lddw : n0);
      q.g.ldc = (uint32_t)m.lddw;
      q.rows_out = q.g.M;
      q.cols_out = q.g.N;
      q.raw = acc + sum_bytes / 4;
      s = terms_product(h, dw_split > 1 ? LM_TERMS_RAW_T : LM_TERMS_ROWS, q, false, tw ? zt : xt, tw ? xt : zt, tw, !tw, dw_tile,
                        dw_split);
      if (s != BWPP_HIP_OK) return s;
      if (dw_split > 1) {
        BwppXentRowArgs f = {};
        f.src = q.raw;
        f.nparts = dw_split;
        f.rows = q.g.M;
        f.cols = q.g.N;
        f.y = q.g.c;
        f.ldy = m.lddw;
        if ((s = bwpp_hip_launch_lm(h, LM_XENT_ROUND, xent_grid(h, f.rows), xent_columns(f.rows, f.cols), 256, &f)) != BWPP_HIP_OK) return s;
      }
    }
  }
  if (!dx) return BWPP_HIP_OK;
  r.y = dx;
  r.ldy = m.lddx;
  r.cols = p.dim;
  r.src = acc;
  r.nparts = split;
  return bwpp_hip_launch_lm(h, LM_XENT_ROUND, xent_grid(h, T), xent_columns(T, p.dim), 256, &r);
}

}  // namespace

extern "C" BwppHipStatus bwpp_hip_dispatch_linear_xent(BwppHip *h, const void *x, const void *w,
                                                       const int32_t *targets, float *loss, float *lse, float *sums,
                                                       BwppLinearXentParams p) {
  const char *what = "linear_xent";
  if (p.rows && (!x || !w || !targets || (!loss && !lse && !sums)))
    return bwpp_hip_set_error(h, BWPP_HIP_ERR_INVALID_ARG, "%s: NULL x, w or targets, or no output", what);
  XentMatrices m;
  BwppHipStatus s = xent_prepare(h, what, p, m);
  if (s != BWPP_HIP_OK) return s;
  const uint64_t T = p.rows, es = p.dtype == BWPP_HIP_BF16 ? 2 : 4;
  {
    const Block in[3] = {{x, T, p.dim * es, m.ldx * es}, {w, m.wrows, m.wcols * es, m.ldw * es}, {targets, 1, T * 4, T * 4}};
    const Block out[3] = {{loss, 1, T * 4, T * 4}, {lse, 1, T * 4, T * 4}, {sums, 1, 8, 8}};
    for (int i = 0; i < 3; ++i) {
      for (const Block &b : in)
        if (meet(out[i], b, 1)) return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: an output overlaps an input", what);
      for (int j = 0; j < i; ++j)
        if (meet(out[i], out[j], 1)) return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: two outputs overlap", what);
    }
  }
  if ((s = bwpp_hip_enter(h)) != BWPP_HIP_OK) return s;
  BwppXentRowArgs r = {};
  r.target = targets;
  r.rows = p.rows;
  r.vocab = p.vocab;
  r.loss = loss;
  r.lse = lse;
  r.sums = sums;
  r.scale = p.scale != 0.0f ? p.scale : 1.0f;
  if (T == 0) return sums ? bwpp_hip_launch_lm(h, LM_XENT_SUMS, 1, 1, 1024, &r) : BWPP_HIP_OK;
  // More rows than one block joins: the sums are taken from the losses.
  const bool own_loss = sums && !loss && T > 64;
  const uint64_t loss_bytes = own_loss ? up(T * 4, 256) : 0, zt_bytes = up(T * 4, 256);
  void *ws = nullptr;
  if (p.dtype == BWPP_HIP_BF16) {
    BwppXentArgs a = {};
    a.g.a = x;
    a.g.b = w;
    a.g.M = p.rows;
    a.g.N = p.vocab;
    a.g.K = p.dim;
    a.g.lda = (uint32_t)m.ldx;
    a.g.ldb = (uint32_t)m.ldw;
    a.target = targets;
    a.vocab = p.vocab;
    a.scale = r.scale;
    const XentTile tile = xent_tile(h, a.g, p.trans_w != 0, false);
    r.nparts = xent_tiles_n(h, a.g, tile);
    if ((s = bwpp_hip_take_workspace(h, zt_bytes + loss_bytes + (uint64_t)r.nparts * T * 8, &ws)) != BWPP_HIP_OK) return s;
    a.zt = static_cast<float *>(ws);
    a.part = reinterpret_cast<float *>(static_cast<unsigned char *>(ws) + zt_bytes + loss_bytes);
    r.zt = a.zt;
    r.part = a.part;
    if ((s = xent_logits(h, LM_XENT_STATS, a, p.trans_w != 0, tile)) != BWPP_HIP_OK) return s;
  } else if (xent_in_terms(h, p, m, false)) {
    if ((s = terms_stats(h, static_cast<const float *>(x), static_cast<const float *>(w), p, m, zt_bytes + loss_bytes, r, ws)) !=
        BWPP_HIP_OK)
      return s;
  } else {
    const uint32_t piece = xent_piece(T, p.vocab, 4);
    const uint64_t npieces = (p.vocab + (uint64_t)piece - 1) / piece;
    const uint64_t part_bytes = up(npieces * T * 8, 256), z_bytes = up(T * up(piece, 4) * 4, 256);
    const uint64_t held = zt_bytes + loss_bytes + part_bytes + z_bytes;
    if ((s = bwpp_hip_take_workspace(h, held + kXentSplitRoom, &ws)) != BWPP_HIP_OK) return s;
    Hold hold(h, held);
    unsigned char *base = static_cast<unsigned char *>(ws);
    r.zt = reinterpret_cast<float *>(base);
    float *part = reinterpret_cast<float *>(base + zt_bytes + loss_bytes);
    float *z = reinterpret_cast<float *>(base + zt_bytes + loss_bytes + part_bytes);
    for (uint64_t i = 0; i < npieces; ++i) {
      const uint32_t n0 = (uint32_t)(i * piece), n = std::min(piece, p.vocab - n0);
      if ((s = xent_logits_f32(h, static_cast<const float *>(x), static_cast<const float *>(w), z, n0, n, p, m)) != BWPP_HIP_OK)
        return s;
      r.src = z;
      r.lds = up(n, 4);
      r.cols = n;
      r.n_base = n0;
      r.part = part + i * T * 2;
      if ((s = bwpp_hip_launch_lm(h, LM_XENT_STATS_F32, xent_grid(h, T), 1, 256, &r)) != BWPP_HIP_OK) return s;
    }
    r.part = part;
    r.nparts = (uint32_t)npieces;
  }
  if (own_loss) r.loss = reinterpret_cast<float *>(static_cast<unsigned char *>(ws) + zt_bytes);
  r.lanes = 1;
  while (r.lanes < 64 && r.lanes < T) r.lanes *= 2;
  if ((s = bwpp_hip_launch_lm(h, LM_XENT_JOIN, (T + r.lanes - 1) / r.lanes, 1, 1024, &r)) != BWPP_HIP_OK) return s;
  return sums && T > 64 ? bwpp_hip_launch_lm(h, LM_XENT_SUMS, 1, 1, 1024, &r) : BWPP_HIP_OK;
}

extern "C" BwppHipStatus bwpp_hip_dispatch_linear_xent_grad(BwppHip *h, const void *x, const void *w,
                                                            const int32_t *targets, const float *lse,
                                                            const float *dloss, void *dx, void *dw,
                                                            BwppLinearXentParams p) {
  const char *what = "linear_xent_grad";
  if (p.rows && (!x || !w || !targets || !lse || (!dx && !dw)))
    return bwpp_hip_set_error(h, BWPP_HIP_ERR_INVALID_ARG, "%s: NULL x, w, targets or lse, or no output", what);
  XentMatrices m;
  BwppHipStatus s = xent_prepare(h, what, p, m);
  if (s != BWPP_HIP_OK) return s;
  const bool bf16 = p.dtype == BWPP_HIP_BF16, tw = p.trans_w != 0;
  const uint64_t T = p.rows, es = bf16 ? 2 : 4, D = p.dim;
  {
    const uint64_t nd = p.dloss_scalar ? 4 : T * 4;
    const Block in[5] = {{x, T, D * es, m.ldx * es}, {w, m.wrows, m.wcols * es, m.ldw * es}, {targets, 1, T * 4, T * 4},
                         {lse, 1, T * 4, T * 4}, {dloss, 1, nd, nd}};
    const Block out[2] = {{dx, T, D * es, m.lddx * es}, {dw, m.wrows, m.wcols * es, m.lddw * es}};
    for (const Block &o : out)
      for (const Block &b : in)
        if (meet(o, b, 1)) return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: an output overlaps an input", what);
    if (meet(out[0], out[1], 1)) return bwpp_hip_set_error(h, BWPP_HIP_ERR_ALIAS, "%s: dx overlaps dw", what);
  }
  if ((s = bwpp_hip_enter(h)) != BWPP_HIP_OK) return s;
  BwppXentRowArgs r = {};
  r.target = targets;
  r.rows = p.rows;
  r.vocab = p.vocab;
  r.scale = p.scale != 0.0f ? p.scale : 1.0f;
  r.dloss = dloss;
  r.dloss_scalar = p.dloss_scalar;
  r.lse_in = lse;
  if (T == 0) {
    if (!dw) return BWPP_HIP_OK;
    r.y = dw;
    r.rows = (uint32_t)m.wrows;
    r.cols = (uint32_t)(m.wcols * (es / 2));  // (fewer than 2^31 columns)
    r.ldy = m.lddw * (es / 2);
    return bwpp_hip_launch_lm(h, LM_XENT_CLEAR, xent_grid(h, m.wrows), xent_columns(m.wrows, r.cols), 256, &r);
  }
  if (!bf16 && xent_in_terms(h, p, m, true))
    return terms_grad(h, static_cast<const float *>(x), static_cast<const float *>(w), static_cast<float *>(dx),
                      static_cast<float *>(dw), p, m, r);
  // bf16: dx is summed in fp32 over pieces, and over planes of K ranges: on 256-wide
  // tiles where they keep half of the CUs busy with a few planes, else on the tiles
  // and ranges that are modelled fastest (4096 x 2048 from 32768 columns: 645 us as
  // one product, 515 on 256-wide tiles and two planes).
  const uint32_t piece = xent_piece(T, p.vocab, es);
  const uint64_t npieces = (p.vocab + (uint64_t)piece - 1) / piece, dx_tiles = ((T + 255) / 256) * ((D + 255) / 256);
  bool wide = bf16 && dx && T > 128 && piece >= 32 && on16(w) && m.ldw % 8 == 0 && (!tw || D % 8 == 0) &&
              256ull * std::max<uint64_t>(piece + 8ull, m.ldw) < (1ull << 31);
  uint32_t split = 1;
  while (wide && split < 8 && dx_tiles * split * 2 <= cus_of(h) && piece / (split * 2) >= 2048) split *= 2;
  wide = wide && dx_tiles * split * 2 >= cus_of(h);
  const bool sums = bf16 && dx && piece >= 8;  // (a chunk of dz)
  XentTile dx_tile = XT_P;
  if (sums && !wide) {
    BwppGemmArgs g = {};
    g.b = w;
    g.M = p.rows;
    g.N = p.dim;
    g.K = piece;
    g.lda = (uint32_t)up(piece, 8);
    g.ldb = (uint32_t)m.ldw;
    dx_tile = xent_tile(h, g, !tw, true, &split);
  }
  if (split > 1) {  // as xent_product cuts the ranges
    const uint32_t k = wide ? piece / 32 * 32 : piece, range = (uint32_t)up((k + split - 1) / split, 128);
    split = (k + range - 1) / range;
  }
  // dW on 256-wide tiles where they keep half of the CUs busy, or, K (tokens) being
  // short, an eighth (17 x 320 x 768 training 34 us on those, 28 to 32 on the others;
  // 256 x 1024 x 2048 48, 39 to 43; at 36 tiles, 210 x 201 x 9001, still 64 and 58,
  // but a test names the kernel there); else on the tiles and K ranges that are
  // modelled fastest, several ranges summed from planes.  (Rows that 32-bit offsets do
  // not span: dispatch_matmul's, without the targets' remainders.)
  const bool dw_fits = bf16 && 256ull * std::max<uint64_t>(piece + 8ull, D + 8) < (1ull << 31);
  const uint64_t dw_tiles = ((piece + 255ull) / 256) * ((D + 255) / 256);
  const bool dw_wide = dw_fits && (dw_tiles * 2 >= cus_of(h) || (T <= 256 && dw_tiles * 8 > cus_of(h)));
  const bool dw_ring = dw && dw_fits && !dw_wide;
  uint32_t dw_split = 1;
  XentTile dw_tile = XT_P;
  if (dw_ring) {
    BwppGemmArgs g = {};
    g.M = (uint32_t)(tw ? up(piece, 8) : up(D, 8));
    g.N = (uint32_t)(tw ? up(D, 8) : up(piece, 8));
    g.K = (uint32_t)up(T, 32);
    g.lda = g.M;
    g.ldb = g.N;
    dw_tile = xent_tile(h, g, false, true, &dw_split);
    const uint32_t range = dw_split > 1 ? (uint32_t)up((g.K + (uint64_t)dw_split - 1) / dw_split, 128) : g.K;
    dw_split = (g.K + range - 1) / range;  // as xent_product cuts them
  }
  // (rows of x's copy and of dz up to a multiple of 32, zeros: dW's K)
  const uint64_t unit = bf16 ? 8 : 4, ldxc = up(D, unit), ldz = up(piece, unit), Tu = bf16 ? up(T, 32) : T;
  const uint64_t x_bytes = dw ? up(Tu * ldxc * es, 256) : 0, z_bytes = up(Tu * ldz * es, 256);
  const uint64_t sum_bytes = sums ? up(split * T * D * 4, 256) : 0, rest_bytes = bf16 ? up(T * 4, 256) : 0;
  const uint64_t dw_bytes = dw_split > 1 ? dw_split * (uint64_t)piece * D * 4 : 0;
  const uint64_t held = x_bytes + z_bytes + sum_bytes + rest_bytes + dw_bytes;
  void *ws = nullptr;
  if ((s = bwpp_hip_take_workspace(h, held + (bf16 ? 0 : kXentSplitRoom), &ws)) != BWPP_HIP_OK) return s;
  Hold hold(h, held);
  unsigned char *base = static_cast<unsigned char *>(ws);
  void *xc = base, *z = base + x_bytes;
  float *acc = reinterpret_cast<float *>(base + x_bytes + z_bytes);
  // What rounding leaves of the targets' dz, for the kernels that add it: dx from
  // planes, and dW's.
  float *rest = reinterpret_cast<float *>(base + x_bytes + z_bytes + sum_bytes);
  auto at = [&](const void *ptr, uint64_t elems) {
    return static_cast<const unsigned char *>(ptr) + elems * es;
  };
  if (dw) {
    r.x = x;
    r.y = xc;
    r.ldx = m.ldx;
    r.ldy = ldxc;
    r.cols = p.dim;
    r.rows_up = (uint32_t)Tu;
    if ((s = bwpp_hip_launch_lm(h, LM_XENT_COPY + bf16, xent_grid(h, Tu), 1, 256, &r)) != BWPP_HIP_OK) return s;
  }
  for (uint64_t i = 0; i < npieces; ++i) {
    const uint32_t n0 = (uint32_t)(i * piece), n = std::min(piece, p.vocab - n0);
    const uint64_t ldp = up(n, unit);
    const void *wp = at(w, tw ? n0 * m.ldw : n0);
    if (bf16) {
      BwppXentArgs a = {};
      a.g.a = x;
      a.g.b = wp;
      a.g.M = p.rows;
      a.g.N = n;
      a.g.K = p.dim;
      a.g.lda = (uint32_t)m.ldx;
      a.g.ldb = (uint32_t)m.ldw;
      a.target = targets;
      a.lse = lse;
      a.dloss = dloss;
      a.dloss_scalar = p.dloss_scalar;
      a.n_base = n0;
      a.vocab = p.vocab;
      a.scale = r.scale;
      a.dl = static_cast<uint16_t *>(z);
      a.ldl = (uint32_t)ldp;
      a.rows_up = (uint32_t)Tu;
      a.rest = rest;
      if ((s = xent_logits(h, LM_XENT_GRAD, a, tw, xent_tile(h, a.g, tw, false))) != BWPP_HIP_OK) return s;
    } else {
      if ((s = xent_logits_f32(h, static_cast<const float *>(x), static_cast<const float *>(w), static_cast<float *>(z), n0,
                               n, p, m)) != BWPP_HIP_OK)
        return s;
      r.y = z;
      r.ldy = ldp;
      r.cols = n;
      r.n_base = n0;
      if ((s = bwpp_hip_launch_lm(h, LM_XENT_GRAD_F32, xent_grid(h, T), 1, 256, &r)) != BWPP_HIP_OK) return s;
    }
    if (dx && sums) {
      BwppXentArgs a = {};
      a.g.a = z;
      a.g.b = wp;
      a.g.M = p.rows;
      a.g.N = p.dim;
      a.g.K = n;
      a.g.lda = (uint32_t)ldp;
      a.g.ldb = (uint32_t)m.ldw;
      a.raw = acc;
      a.accumulate = i > 0;
      if (!wide) {
        // (the last piece may be cut for other loads, never for more ranges)
        const XentTile tile = n == piece ? dx_tile : xent_tile(h, a.g, !tw, true);
        if ((s = xent_product(h, LM_XENT_RAW, a, !tw, tile, split)) != BWPP_HIP_OK) return s;
      } else {  // K in steps of 32, what is left of it on other tiles
        BwppXentArgs rest = a;
        a.g.K = n / 32 * 32;
        if (a.g.K && (s = xent_product(h, LM_XENT_RAW, a, !tw, XT_P, split)) != BWPP_HIP_OK) return s;
        if (n % 32) {
          rest.g.K = n % 32;
          rest.g.a = static_cast<const uint16_t *>(rest.g.a) + a.g.K;
          rest.g.b = static_cast<const uint16_t *>(rest.g.b) + (tw ? (uint64_t)a.g.K * m.ldw : a.g.K);
          rest.accumulate = i > 0 || a.g.K;
          if ((s = xent_product(h, LM_XENT_RAW, rest, !tw, xent_tile(h, rest.g, !tw, true), 1)) != BWPP_HIP_OK) return s;
        }
      }
    } else if (dx) {
      BwppMatmulParams g = {};
      g.M = p.rows;
      g.N = p.dim;
      g.K = n;
      g.lda = (uint32_t)ldp;
      g.ldb = (uint32_t)m.ldw;
      g.ldc = (uint32_t)m.lddx;
      g.dtype = p.dtype;
      g.trans_b = tw ? 0u : 1u;
      BwppHipFusionParams f = {};
      f.kind = i > 0 ? BWPP_HIP_FUSE_RESIDUAL : BWPP_HIP_FUSE_NONE;
      f.ld_aux = g.ldc;
      s = bwpp_hip_dispatch_matmul_fused(h, z, wp, dx, nullptr, i > 0 ? static_cast<const float *>(dx) : nullptr, nullptr, g, f);
      if (s != BWPP_HIP_OK) return s;
    }
    void *dwp = dw ? const_cast<unsigned char *>(at(dw, tw ? n0 * m.lddw : n0)) : nullptr;
    if (dw && (dw_wide || dw_ring)) {
      BwppXentArgs a = {};
      a.g.a = tw ? z : xc;
      a.g.b = tw ? xc : z;
      a.g.c = dwp;
      a.g.M = (uint32_t)(tw ? ldp : ldxc);
      a.g.N = (uint32_t)(tw ? ldxc : ldp);
      a.g.K = (uint32_t)Tu;
      a.g.lda = a.g.M;
      a.g.ldb = a.g.N;
      a.g.ldc = (uint32_t)m.lddw;
      a.rows_out = tw ? n : p.dim;
      a.cols_out = tw ? p.dim : n;
      a.target = targets;
      a.vocab = p.vocab;
      a.n_base = n0;
      a.rest = rest;
      a.rows = p.rows;
      a.x_is_a = !tw;
      a.raw = reinterpret_cast<float *>(base + x_bytes + z_bytes + sum_bytes + rest_bytes);
      const int ring = (dw_tile - XT_R32) / 2 - dw_tile;  // XT_R32, XT_R64, XT_R128 as 0, 1, 2
      s = xent_product(h, !dw_ring ? LM_XENT_ROWS : (dw_split > 1 ? LM_XENT_ROW_SUMS : LM_XENT_ROWS_RING) + ring, a, false,
                       dw_tile, dw_split);
      if (s != BWPP_HIP_OK) return s;
      if (dw_split > 1) {
        BwppXentRowArgs f = {};
        f.src = a.raw;
        f.nparts = dw_split;
        f.rows = a.rows_out;
        f.cols = a.cols_out;
        f.y = dwp;
        f.ldy = m.lddw;
        if ((s = bwpp_hip_launch_lm(h, LM_XENT_ROUND + 1, xent_grid(h, f.rows), xent_columns(f.rows, f.cols), 256, &f)) != BWPP_HIP_OK) return s;
      }
    } else if (dw) {
      BwppMatmulParams g = {};
      g.K = p.rows;
      g.M = tw ? n : p.dim;
      g.N = tw ? p.dim : n;
      g.lda = (uint32_t)(tw ? ldp : ldxc);
      g.ldb = (uint32_t)(tw ? ldxc : ldp);
      g.ldc = (uint32_t)m.lddw;
      g.dtype = p.dtype;
      g.trans_a = 1;
      if ((s = bwpp_hip_dispatch_matmul(h, tw ? z : xc, tw ? xc : z, dwp, nullptr, g)) != BWPP_HIP_OK) return s;
    }
  }
  if (!dx) return BWPP_HIP_OK;
  r.y = dx;
  r.ldy = m.lddx;
  r.cols = p.dim;
  if (!sums) return bwpp_hip_launch_lm(h, LM_XENT_ZERO + bf16, xent_grid(h, T), 1, 256, &r);
  r.src = acc;
  r.nparts = split;
  r.rest = rest;
  r.w = w;
  r.ldw = m.ldw;
  if (tw) return bwpp_hip_launch_lm(h, LM_XENT_ROUND + 1, xent_grid(h, T), xent_columns(T, p.dim), 256, &r);
  r.lanes = T >= 1024 ? 64 : 8;
  const uint64_t blocks = up((D + 31) / 32, 8) * ((T + r.lanes - 1) / r.lanes);
  if (blocks * 256 > 0xffffffffull) return bwpp_hip_set_error(h, BWPP_HIP_ERR_UNSUPPORTED, "%s: too many elements", what);
  return bwpp_hip_launch_lm(h, LM_XENT_ROUND + 2, blocks, 1, 256, &r);
}

// Operators of libbwpp_hip for a serving loop: a paged cache of keys and values
// (append with rotary positions, attention, accepted drafts) and rules on
// logits.  Argument checks, launch geometry and the choice of a kernel; the
// kernels are kv_append.h, kv_attention.h and logit_rules.h.
#include "bwpp_hip.h"
#include "internal.h"
#include "rowset.h"

#include <algorithm>
#include <cmath>

#include "../kargs.h"

namespace {

enum CacheKernel {
  CK_APPEND_BF16,                      // [interleaved][chunk 8, 4, 1]
  CK_APPEND_F32 = CK_APPEND_BF16 + 6,  // [interleaved][chunk 4, 1]
  CK_KEEP = CK_APPEND_F32 + 4,         // chunks of 16, 4, 2 bytes
  CK_ATTEND = CK_KEEP + 3,             // [bf16][dim up to 64, 128, 192, 256]
  CK_ATTEND_ROWS = CK_ATTEND + 8,      // [bf16][dim up to 32, 64, .. 256]
  CK_ATTEND_FEW = CK_ATTEND_ROWS + 16, // [kFlashDims]
  CK_ATTEND_R128 = CK_ATTEND_FEW + 7,  // [kFlashDims]
  CK_ATTEND_R256 = CK_ATTEND_R128 + 7, // [kFlashDims up to 128]
  CK_JOIN_F32 = CK_ATTEND_R256 + 4,    // tiles of 16, 128 rows
  CK_JOIN_BF16 = CK_JOIN_F32 + 2,      // of 16, 32, 128, 256
  CK_RULES = CK_JOIN_BF16 + 4,         // [x bf16][y bf16]
  CK_COUNT = CK_RULES + 4
};

}  // namespace

const char *const bwpp_hip_cache_kernels[] = {
    "bwpp_cache_append_bf16_half_8",
    "bwpp_cache_append_bf16_half_4",
    "bwpp_cache_append_bf16_half_1",
    "bwpp_cache_append_bf16_inter_8",
    "bwpp_cache_append_bf16_inter_4",
    "bwpp_cache_append_bf16_inter_1",
    "bwpp_cache_append_f32_half_4",
    "bwpp_cache_append_f32_half_1",
    "bwpp_cache_append_f32_inter_4",
    "bwpp_cache_append_f32_inter_1",
    "bwpp_cache_keep_16",
    "bwpp_cache_keep_4",
    "bwpp_cache_keep_2",
    "bwpp_cache_attend_f32_d64",
    "bwpp_cache_attend_f32_d128",
    "bwpp_cache_attend_f32_d192",
    "bwpp_cache_attend_f32_d256",
    "bwpp_cache_attend_bf16_d64",
    "bwpp_cache_attend_bf16_d128",
    "bwpp_cache_attend_bf16_d192",
    "bwpp_cache_attend_bf16_d256",
    "bwpp_cache_attend_f32_rows_d32",
    "bwpp_cache_attend_f32_rows_d64",
    "bwpp_cache_attend_f32_rows_d96",
    "bwpp_cache_attend_f32_rows_d128",
    "bwpp_cache_attend_f32_rows_d160",
    "bwpp_cache_attend_f32_rows_d192",
    "bwpp_cache_attend_f32_rows_d224",
    "bwpp_cache_attend_f32_rows_d256",
    "bwpp_cache_attend_bf16_rows_d32",
    "bwpp_cache_attend_bf16_rows_d64",
    "bwpp_cache_attend_bf16_rows_d96",
    "bwpp_cache_attend_bf16_rows_d128",
    "bwpp_cache_attend_bf16_rows_d160",
    "bwpp_cache_attend_bf16_rows_d192",
    "bwpp_cache_attend_bf16_rows_d224",
    "bwpp_cache_attend_bf16_rows_d256",
    "bwpp_cache_attend_few_d64",
    "bwpp_cache_attend_few_d80",
    "bwpp_cache_attend_few_d96",
    "bwpp_cache_attend_few_d128",
    "bwpp_cache_attend_few_d160",
    "bwpp_cache_attend_few_d192",
    "bwpp_cache_attend_few_d256",
    "bwpp_cache_attend_r128_d64",
    "bwpp_cache_attend_r128_d80",
    "bwpp_cache_attend_r128_d96",
    "bwpp_cache_attend_r128_d128",
    "bwpp_cache_attend_r128_d160",
    "bwpp_cache_attend_r128_d192",
    "bwpp_cache_attend_r128_d256",
    "bwpp_cache_attend_r256_d64",
    "bwpp_cache_attend_r256_d80",
    "bwpp_cache_attend_r256_d96",
    "bwpp_cache_attend_r256_d128",
    "bwpp_cache_join_f32_16",
    "bwpp_cache_join_f32_128",
    "bwpp_cache_join_bf16_16",
    "bwpp_cache_join_bf16_32",
    "bwpp_cache_join_bf16_128",
    "bwpp_cache_join_bf16_256",
    "bwpp_logit_rules_f32",
    "bwpp_logit_rules_f32_bf16",
    "bwpp_logit_rules_bf16_f32",
    "bwpp_logit_rules_bf16",
};
const int bwpp_hip_cache_kernel_count = (int)(sizeof(bwpp_hip_cache_kernels) / sizeof(bwpp_hip_cache_kernels[0]));
static_assert(sizeof(bwpp_hip_cache_kernels) / sizeof(bwpp_hip_cache_kernels[0]) == CK_COUNT, "kernel names");

namespace {

// Head dims of the bf16 matrix-core kernels (kv_flash.h).
const uint32_t kFlashDims[] = {64, 80, 96, 128, 160, 192, 256};

BwppHipFault invalid(const char *why) { return {BWPP_HIP_ERR_INVALID_ARG, why}; }
BwppHipFault unsupported(const char *why) { return {BWPP_HIP_ERR_UNSUPPORTED, why}; }

uint32_t cus_of(const BwppHip *h) {
  const int n = bwpp_hip_device_cus(h);
  return n > 0 ? (uint32_t)n : 256u;
}

// A stretch of memory of a small operand.
struct Span {
  const void *p;
  uint64_t bytes;
};
bool meet(const RowSet &r, const Span &s, uint64_t es) {
  return r.p && s.p && s.bytes && bwpp_hip_blocks_overlap(r.p, 1, r.span() * es, 0, s.p, 1, s.bytes, 0, 1);
}
bool meet(const Span &a, const Span &b) {
  return a.p && b.p && a.bytes && b.bytes && bwpp_hip_blocks_overlap(a.p, 1, a.bytes, 0, b.p, 1, b.bytes, 0, 1);
}

// The cache's shape: strides with their defaults, a pool's rows.
struct Cache {
  uint64_t page_s, tok_s, head_s, ld_table, capacity, es;
  uint32_t shift;
  RowSet pool(const void *p, const BwppCacheParams &c) const {
    return {p, tok_s, head_s, page_s, c.pages, c.heads, c.page_tokens, c.dim};
  }
};

BwppHipFault check_cache(const BwppCacheParams &p, Cache &c) {
  if (p.dtype > BWPP_HIP_BF16) return invalid("unknown dtype");
  if (p.page_tokens == 0 || (p.page_tokens & (p.page_tokens - 1))) return invalid("page_tokens must be a power of two");
  if (p.heads == 0 || p.dim == 0) return invalid("no key heads or dim");
  if (p.q_heads % p.heads) return invalid("q_heads must be a multiple of heads");
  if (p.ld_table != 0 && p.ld_table < p.max_pages) return invalid("ld_table smaller than max_pages");
  c.es = p.dtype == BWPP_HIP_BF16 ? 2 : 4;
  c.tok_s = p.token_stride ? p.token_stride : p.dim;
  c.head_s = p.head_stride ? p.head_stride : p.page_tokens * c.tok_s;
  c.page_s = p.page_stride ? p.page_stride : p.heads * c.head_s;
  c.ld_table = p.ld_table ? p.ld_table : p.max_pages;
  c.shift = (uint32_t)__builtin_ctz(p.page_tokens);
  c.capacity = std::min<uint64_t>((uint64_t)p.max_pages << c.shift, 0x7fffffffull);
  if (p.batch > (1u << 24) || (uint64_t)p.tokens * std::max(1u, p.q_heads) >= (1ull << 31) || p.heads > (1u << 16) ||
      p.dim > 4096 || p.q_heads > (1u << 16))
    return unsupported("batch above 2^24, tokens q_heads of 2^31, heads above 2^16 or dim above 4096");
  const long double span = (long double)p.pages * c.page_s + (long double)p.heads * c.head_s + (long double)p.page_tokens * c.tok_s;
  if (span > 1152921504606846976.0L) return unsupported("strides of a pool that reach 2^60 elements");
  return {BWPP_HIP_OK, nullptr};
}

BwppRotaryParams rotation(const BwppCacheAppendParams &p) {
  BwppRotaryParams r = {};
  r.tokens = p.cache.tokens;
  r.q_heads = p.cache.q_heads;
  r.k_heads = p.cache.heads;
  r.dim = p.cache.dim;
  r.rot_dim = p.rot_dim;
  r.layout = p.layout;
  r.dtype = p.cache.dtype;
  r.scaling = p.scaling;
  r.base = p.base;
  r.factor = p.factor;
  r.low_turns = p.low_turns;
  r.high_turns = p.high_turns;
  r.context = p.context;
  r.magnitude = p.magnitude;
  return r;
}

BwppHipFault check_append(const BwppCacheAppendParams &p, Cache &c) {
  const BwppHipFault f = check_cache(p.cache, c);
  if (f.why || p.no_rotation) return f;
  return bwpp_hip_check_rotary(rotation(p));
}

BwppHipFault check_attention(const BwppCacheAttentionParams &p, bool mask, Cache &c) {
  const BwppHipFault f = check_cache(p.cache, c);
  if (f.why) return f;
  if (p.cache.q_heads == 0) return invalid("no query heads");
  if (!std::isfinite(p.scale)) return invalid("scale must be finite");
  if (mask && p.mask_words == 0) return invalid("a mask without words");
  if (p.cache.dim > 256) return unsupported("dim above 256");
  return f;
}

BwppHipFault check_keep(const BwppCacheKeepParams &p, Cache &c) {
  BwppCacheParams cp = p.cache;
  cp.tokens = 0;
  cp.q_heads = 0;
  const BwppHipFault f = check_cache(cp, c);
  if (f.why) return f;
  if (p.ld_kept != 0 && p.ld_kept < p.max_kept) return invalid("ld_kept smaller than max_kept");
  return f;
}

void fill(BwppCacheArgs &a, const BwppCacheParams &p, const Cache &c, const void *k, const void *v,
          const int32_t *table, const int32_t *starts, const int32_t *held) {
  a.k = const_cast<void *>(k);
  a.v = const_cast<void *>(v);
  a.table = table;
  a.starts = starts;
  a.held = held;
  a.page_s = c.page_s;
  a.tok_s = c.tok_s;
  a.head_s = c.head_s;
  a.ld_table = c.ld_table;
  a.pages = p.pages;
  a.page_shift = c.shift;
  a.capacity = (uint32_t)c.capacity;
  a.batch = p.batch;
  a.tokens = p.tokens;
  a.heads = p.heads;
  a.dim = p.dim;
}

// Rows of the new tokens: [tokens][heads][dim] where strides are zero.
RowSet token_rows(const void *p, uint64_t tokens, uint64_t heads, uint64_t dim, uint64_t ld, uint64_t head_stride) {
  const uint64_t hs = head_stride ? head_stride : dim;
  return {heads ? p : nullptr, ld ? ld : heads * dim, hs, 0, 1, heads ? heads : 1, tokens, dim};
}
// Whether a token's stride is too short for a row, or one row lies in another.
bool bad_rows(const RowSet &r, bool written) {
  if (!r.p) return false;
  if (r.tokens > 1 && r.ts < r.dim) return true;
  return written && !disjoint_rows(r);
}

}  // namespace

BwppHipFault bwpp_hip_check_cache_append(const BwppCacheAppendParams &p) {
  Cache c = {};
  return check_append(p, c);
}
BwppHipFault bwpp_hip_check_cache_attention(const BwppCacheAttentionParams &p, bool mask) {
  Cache c = {};
  return check_attention(p, mask, c);
}
BwppHipFault bwpp_hip_check_cache_keep(const BwppCacheKeepParams &p) {
  Cache c = {};
  return check_keep(p, c);
}
BwppHipFault bwpp_hip_check_logit_rules(const BwppLogitRulesParams &p) {
  if (p.dtype_x > BWPP_HIP_BF16 || p.dtype_y > BWPP_HIP_BF16) return invalid("unknown dtype");
  if ((p.ldx && p.ldx < p.vocab) || (p.ldy && p.ldy < p.vocab) || (p.ld_bias && p.ld_bias < p.vocab) ||
      (p.ld_mask && p.ld_mask < ((uint64_t)p.vocab + 31) / 32))
    return invalid("row stride smaller than the row");
  if (p.vocab > 0x7fffffffu || p.history > 0x7fffffffu) return unsupported("vocab or history of 2^31 or more");
  return {BWPP_HIP_OK, nullptr};
}

// ------------------------------------------------------------------ append

extern "C" BwppHipStatus bwpp_hip_dispatch_cache_append(BwppHip *h, const void *q, const void *k, const void *v,
                                                        const int32_t *positions, const int32_t *table,
                                                        const int32_t *starts, const int32_t *held, void *qo,
                                                        void *k_cache, void *v_cache, BwppCacheAppendParams p) {
  auto bad = [&](BwppHipStatus s, const char *why) { return bwpp_hip_set_error(h, s, "cache_append: %s", why); };
  const BwppCacheParams &cp = p.cache;
  Cache c = {};
  const BwppHipFault fault = check_append(p, c);
  if (fault.why) return bad(fault.status, fault.why);
  if (cp.tokens == 0 || cp.batch == 0) return bwpp_hip_enter(h);
  const bool pool = cp.pages && cp.max_pages;  // somewhere to write
  if ((cp.q_heads && (!q || !qo)) || !k || !v || !starts || !held || (pool && (!table || !k_cache || !v_cache)))
    return bad(BWPP_HIP_ERR_INVALID_ARG, "NULL operand");
  const uint64_t T = cp.tokens, d = cp.dim, es = c.es;
  const RowSet sq = token_rows(q, T, cp.q_heads, d, p.ldq, p.q_head_stride);
  const RowSet sk = token_rows(k, T, cp.heads, d, p.ldk, p.k_head_stride);
  const RowSet sv = token_rows(v, T, cp.heads, d, p.ldv, p.v_head_stride);
  const RowSet dq = token_rows(qo, T, cp.q_heads, d, p.ldqo, p.qo_head_stride);
  const RowSet dk = c.pool(pool ? k_cache : nullptr, cp), dv = c.pool(pool ? v_cache : nullptr, cp);
  if (bad_rows(sq, false) || bad_rows(sk, false) || bad_rows(sv, false) || bad_rows(dq, true))
    return bad(BWPP_HIP_ERR_INVALID_ARG, "token stride smaller than the row, or rows of an output overlap");
  if (pool && !disjoint_rows(dk)) return bad(BWPP_HIP_ERR_INVALID_ARG, "rows of a pool overlap");
  const bool in_place = sq.p && same_rows(sq, dq);
  bool alias = (!in_place && meet(dq, sq, es)) || meet(dq, sk, es) || meet(dq, sv, es) || meet(dk, dv, es);
  for (const RowSet *o : {&dk, &dv})
    alias = alias || meet(*o, sq, es) || meet(*o, sk, es) || meet(*o, sv, es) || meet(*o, dq, es);
  const Span small[4] = {{positions, T * 4},
                         {pool ? table : nullptr, ((cp.batch - 1) * c.ld_table + cp.max_pages) * 4},
                         {starts, ((uint64_t)cp.batch + 1) * 4},
                         {held, (uint64_t)cp.batch * 4}};
  for (const RowSet *o : {&dq, &dk, &dv})
    for (const Span &s : small) alias = alias || meet(*o, s, es);
  if (alias) return bad(BWPP_HIP_ERR_ALIAS, "an output overlaps another operand");
  const BwppHipStatus s = bwpp_hip_enter(h);
  if (s != BWPP_HIP_OK) return s;

  BwppCacheAppendArgs a = {};
  fill(a.c, cp, c, k_cache, v_cache, table, starts, held);
  const uint32_t rot = p.no_rotation ? 0u : p.rot_dim ? p.rot_dim : cp.dim;
  bwpp_hip_rotary_args(rotation(p), rot, a.r);
  a.r.q = sq.p;
  a.r.k = k;
  a.r.qo = qo;
  a.r.positions = positions;
  a.r.q_ts = sq.ts, a.r.q_hs = sq.hs;
  a.r.k_ts = sk.ts, a.r.k_hs = sk.hs;
  a.r.qo_ts = dq.ts, a.r.qo_hs = dq.hs;
  a.v_in = v;
  a.v_ts = sv.ts, a.v_hs = sv.hs;
  a.r.heads = cp.q_heads + 2 * cp.heads;
  a.r.copy = in_place ? 0u : 1u;
  const bool bf16 = cp.dtype == BWPP_HIP_BF16, inter = p.layout == BWPP_HIP_ROTARY_INTERLEAVED;
  const uint32_t pick = bf16 ? (a.r.pairs % 8 == 0 ? 0u : a.r.pairs % 4 == 0 ? 1u : 2u) : (a.r.pairs % 4 == 0 ? 0u : 1u);
  const uint32_t chunk = bf16 ? (pick == 0 ? 8u : pick == 1 ? 4u : 1u) : (pick == 0 ? 4u : 1u);
  a.r.tail_chunks = (cp.dim - rot + chunk - 1) / chunk;
  // As rotary: tiles of tokens while eight blocks a CU remain, then groups of heads.
  const uint64_t want = 8ull * cus_of(h);
  const uint32_t most = std::min(64u, std::max(1u, 2048u / std::max(1u, a.r.pairs)));
  a.r.tile = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(most, T), std::max<uint64_t>(1, T / want));
  a.r.hgroup = std::min(a.r.heads, 256u);
  const uint64_t blocks = (T + a.r.tile - 1) / a.r.tile;
  while (a.r.hgroup > 8 && blocks * ((a.r.heads + a.r.hgroup - 1) / a.r.hgroup) * 2 <= want)
    a.r.hgroup = (a.r.hgroup + 1) / 2;
  const uint32_t groups = (a.r.heads + a.r.hgroup - 1) / a.r.hgroup;
  const int index = bf16 ? CK_APPEND_BF16 + (inter ? 3 : 0) + (int)pick : CK_APPEND_F32 + (inter ? 2 : 0) + (int)pick;
  return bwpp_hip_launch_cache(h, index, blocks, groups, 256, &a);
}

// -------------------------------------------------------------------- keep

extern "C" BwppHipStatus bwpp_hip_dispatch_cache_keep(BwppHip *h, void *k_cache, void *v_cache, const int32_t *table,
                                                      const int32_t *held, const int32_t *kept, const int32_t *counts,
                                                      BwppCacheKeepParams p) {
  auto bad = [&](BwppHipStatus s, const char *why) { return bwpp_hip_set_error(h, s, "cache_keep: %s", why); };
  const BwppCacheParams &cp = p.cache;
  Cache c = {};
  const BwppHipFault fault = check_keep(p, c);
  if (fault.why) return bad(fault.status, fault.why);
  if (cp.batch == 0 || p.max_kept == 0 || cp.pages == 0 || cp.max_pages == 0) return bwpp_hip_enter(h);
  if (!k_cache || !v_cache || !table || !held || !kept || !counts) return bad(BWPP_HIP_ERR_INVALID_ARG, "NULL operand");
  const RowSet dk = c.pool(k_cache, cp), dv = c.pool(v_cache, cp);
  if (!disjoint_rows(dk)) return bad(BWPP_HIP_ERR_INVALID_ARG, "rows of a pool overlap");
  const uint64_t ld = p.ld_kept ? p.ld_kept : p.max_kept;
  bool alias = meet(dk, dv, c.es);
  const Span small[4] = {{table, ((cp.batch - 1) * c.ld_table + cp.max_pages) * 4},
                         {held, (uint64_t)cp.batch * 4},
                         {kept, ((cp.batch - 1) * ld + p.max_kept) * 4},
                         {counts, (uint64_t)cp.batch * 4}};
  for (const RowSet *o : {&dk, &dv})
    for (const Span &s : small) alias = alias || meet(*o, s, c.es);
  if (alias) return bad(BWPP_HIP_ERR_ALIAS, "a pool overlaps another operand");
  const BwppHipStatus s = bwpp_hip_enter(h);
  if (s != BWPP_HIP_OK) return s;
  BwppCacheKeepArgs a = {};
  fill(a.c, cp, c, k_cache, v_cache, table, nullptr, held);
  a.kept = kept;
  a.counts = counts;
  a.ld_kept = ld;
  a.max_kept = p.max_kept;
  // Chunks of 16 bytes where every row begins on one, of an element otherwise.
  const uint64_t any = (uintptr_t)k_cache | (uintptr_t)v_cache | c.page_s * c.es | c.tok_s * c.es | c.head_s * c.es | cp.dim * c.es;
  const bool wide = any % 16 == 0;
  a.unit = wide ? (uint32_t)(16 / c.es) : 1u;
  a.chunks = cp.dim / a.unit;
  const uint64_t items = 2ull * cp.heads * a.chunks;
  if (items > 256ull * 65535) return bad(BWPP_HIP_ERR_UNSUPPORTED, "too many heads");
  return bwpp_hip_launch_cache(h, CK_KEEP + (wide ? 0 : c.es == 4 ? 1 : 2), cp.batch, (uint32_t)((items + 255) / 256), 256, &a);
}

// --------------------------------------------------------------- attention

extern "C" BwppHipStatus bwpp_hip_dispatch_cache_attention(BwppHip *h, const void *q, const void *k_cache,
                                                           const void *v_cache, const int32_t *table,
                                                           const int32_t *starts, const int32_t *held,
                                                           const uint32_t *mask, void *o, float *lse,
                                                           BwppCacheAttentionParams p) {
  auto bad = [&](BwppHipStatus s, const char *why) { return bwpp_hip_set_error(h, s, "cache_attention: %s", why); };
  const BwppCacheParams &cp = p.cache;
  Cache c = {};
  const BwppHipFault fault = check_attention(p, mask != nullptr, c);
  if (fault.why) return bad(fault.status, fault.why);
  if (cp.tokens == 0 || cp.batch == 0) return bwpp_hip_enter(h);
  const bool pool = cp.pages && cp.max_pages;
  if (!q || !o || !starts || !held || (pool && (!table || !k_cache || !v_cache)))
    return bad(BWPP_HIP_ERR_INVALID_ARG, "NULL operand");
  const uint64_t T = cp.tokens, d = cp.dim, es = c.es, g = cp.q_heads / cp.heads;
  const RowSet sq = token_rows(q, T, cp.q_heads, d, p.ldq, p.q_head_stride);
  const RowSet so = token_rows(o, T, cp.q_heads, d, p.ldo, p.o_head_stride);
  if (bad_rows(sq, false) || bad_rows(so, true))
    return bad(BWPP_HIP_ERR_INVALID_ARG, "token stride smaller than the row, or rows of the output overlap");
  const RowSet sk = c.pool(pool ? k_cache : nullptr, cp), sv = c.pool(pool ? v_cache : nullptr, cp);
  const Span ls = {lse, T * cp.q_heads * 4};
  const Span small[4] = {{pool ? table : nullptr, ((cp.batch - 1) * c.ld_table + cp.max_pages) * 4},
                         {starts, ((uint64_t)cp.batch + 1) * 4},
                         {held, (uint64_t)cp.batch * 4},
                         {mask, T * p.mask_words * 4}};
  bool alias = meet(so, sq, es) || meet(so, sk, es) || meet(so, sv, es) || meet(so, ls, es) || meet(sq, ls, es) ||
               meet(sk, ls, es) || meet(sv, ls, es);
  for (const Span &s : small) alias = alias || meet(so, s, es) || meet(ls, s);
  if (alias) return bad(BWPP_HIP_ERR_ALIAS, "an output overlaps another operand");
  // bf16 rows of 16-byte chunks (q, keys, values; 8-byte results) take the
  // matrix-core kernels where the lanes' 32-bit offsets in a tile of 64 keys reach.
  int flash = -1;
  const uint64_t chunks = sq.ts | sq.hs | c.tok_s | c.head_s | c.page_s | (uintptr_t)q / 2 | (uintptr_t)k_cache / 2 | (uintptr_t)v_cache / 2;
  if (cp.dtype == BWPP_HIP_BF16 && chunks % 8 == 0 && (so.ts | so.hs | (uintptr_t)o / 2) % 4 == 0 &&
      ((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)o) % 2 == 0 && c.tok_s < (1u << 24) &&
      c.page_s < (1ull << 32))
    for (int i = 0; i < 7; ++i)
      if (kFlashDims[i] == cp.dim) flash = i;
  // Tiles of few rows, whose waves share the keys out, or of more, where each wave
  // has its own: by the rows that a sequence and key head has on average.  16 trees
  // over up to 8000 tokens, 8 key heads of 128: bf16 32 rows 44 us on tiles of 32,
  // 42 of 128, 40 rows 60 and 44; fp32 64 rows 165 on tiles of 16, 179 of 128, 96
  // rows 243 and 187.  bf16, 256 rows over 30000 tokens 52 us on tiles of 128, 43 of
  // 256; 4 x 2000 rows without a past 38 and 30.
  const uint64_t mean = (T + cp.batch - 1) / cp.batch * g;
  const uint32_t rows = flash < 0 ? (mean > 64 ? 128u : 16u) : mean <= 32 ? 32u : mean <= 128 || cp.dim > 128 ? 128u : 256u;
  const uint32_t Dp = (cp.dim + 3) / 4 * 4;
  // Costs (kv_schedule.h) are taken in doubles too: below 2^52; and, whatever starts
  // holds (sequences that overlap each count all rows), in 64 bits with a share more.
  const long double item = (long double)cp.heads * ((long double)g * (c.capacity + 512) + (long double)T * g + 2 * rows);
  if (item * ((long double)T * g / rows + cp.batch) > 4503599627370496.0L ||
      item * ((long double)T * g / rows + 1) * cp.batch > 4611686018427387904.0L)
    return bad(BWPP_HIP_ERR_UNSUPPORTED, "tokens times the longest sequence out of range");
  BwppHipStatus s = bwpp_hip_enter(h);
  if (s != BWPP_HIP_OK) return s;

  BwppCacheAttnArgs a = {};
  fill(a.c, cp, c, k_cache, v_cache, table, starts, held);
  if (!pool) a.c.capacity = 0;
  a.q = q;
  a.o = o;
  a.lse = lse;
  a.mask = mask;
  a.q_ts = sq.ts, a.q_hs = sq.hs, a.o_ts = so.ts, a.o_hs = so.hs;
  a.mask_words = p.mask_words;
  a.group = (uint32_t)g;
  const float scale = p.scale != 0.0f ? p.scale : 1.0f;
  a.scale_log2 = std::fabs(scale) * 1.4426950408889634f;
  a.flip = scale < 0.0f ? 1u : 0u;
  // Blocks as many as are resident at once, the same number on each XCD.
  a.blocks = ((rows == 256 || (rows != 16 && cp.dim > 128) ? 1 : 2) * cus_of(h) + 7) / 8 * 8;
  a.inv_blocks = 1.0 / a.blocks;
  // Up to here an item's keys cost less than its parts and their join: 24
  // sequences of 200 tokens 16.9 us in parts, 11.2 whole, one of 204 12.8 and
  // 10.7, 3 x 550 tokens of 64 : 8 heads 68 and 45 (past 1024 keys parts win: one
  // sequence of 1000 tokens 12.8 in parts, 16 whole; fp32 4 x 416 tokens 300 and 393).
  a.whole_keys = flash < 0 ? 256 : rows == 32 ? 512 : 1024;
  // What starting and ending an item takes, in keys: 128 sequences of up to 2000
  // tokens 57 us with 96, 48 with 192, 49 with 384; 2 x 2048 tokens of prompts over
  // 4000 and 1000 of d = 128 293, 289, 280, of 256 740, 728, 725; fp32 2 x 1024 tokens
  // 257, 268, 284.
  a.item_keys = flash < 0 ? 96 : rows == 32 ? 192 : 384;
  // 256 MiB of keys and values fill the Infinity Cache (costs count some more than the
  // keys).  What is more, and read once, goes past it: 64 steps over 1.9 GB 327 us,
  // past it 293, over 0.5 GB (d = 64) 103 and 91; what it could keep for the next
  // call: 128 steps over 245 MB 48 and 50, 16 trees over 250 MB 60 and 64.  Of one row
  // of pages for all 64, 278 and 280.
  a.large_cost = (320ull << 20) * g / (2 * cp.dim * es);
  // (kv_schedule.h leaves every item whole where no sequence has more keys in its table.)
  const bool parts = c.capacity > a.whole_keys;
  if (parts) {
    void *ws = nullptr;
    s = bwpp_hip_take_workspace(h, (size_t)2 * a.blocks * rows * (Dp + 2) * 4, &ws);
    if (s != BWPP_HIP_OK) return s;
    a.part_o = static_cast<float *>(ws);
    a.part_ml = a.part_o + (size_t)2 * a.blocks * rows * Dp;
  }
  const bool bf16 = cp.dtype == BWPP_HIP_BF16;
  const int attend = flash >= 0    ? flash + (rows == 32 ? CK_ATTEND_FEW : rows == 128 ? CK_ATTEND_R128 : CK_ATTEND_R256)
                     : rows == 128 ? CK_ATTEND_ROWS + (bf16 ? 8 : 0) + (int)((cp.dim - 1) / 32)
                                   : CK_ATTEND + (bf16 ? 4 : 0) + (int)((cp.dim - 1) / 64);
  const int join = bf16 ? CK_JOIN_BF16 + (rows == 16 ? 0 : rows == 32 ? 1 : rows == 128 ? 2 : 3)
                        : CK_JOIN_F32 + (rows == 16 ? 0 : 1);
  s = bwpp_hip_launch_cache(h, attend, a.blocks, 1, rows == 32 ? 128 : rows == 256 ? 512 : 256, &a);
  if (s != BWPP_HIP_OK || !parts) return s;
  return bwpp_hip_launch_cache(h, join, a.blocks - 1, rows <= 32 ? 1 : rows / 64, 256, &a);
}

// ------------------------------------------------------------------- rules

extern "C" BwppHipStatus bwpp_hip_dispatch_logit_rules(BwppHip *h, const void *x, const int32_t *history,
                                                       const int32_t *starts, const int32_t *prompt,
                                                       const float *repetition, const float *presence,
                                                       const float *frequency, const float *bias, const uint32_t *mask,
                                                       void *y, BwppLogitRulesParams p) {
  auto bad = [&](BwppHipStatus s, const char *why) { return bwpp_hip_set_error(h, s, "logit_rules: %s", why); };
  const BwppHipFault fault = bwpp_hip_check_logit_rules(p);
  if (fault.why) return bad(fault.status, fault.why);
  const uint64_t R = p.rows, V = p.vocab, ldx = p.ldx ? p.ldx : V, ldy = p.ldy ? p.ldy : V, words = (V + 31) / 32;
  if (R == 0 || V == 0) return bwpp_hip_enter(h);
  if (!x || !y) return bad(BWPP_HIP_ERR_INVALID_ARG, "NULL x or y");
  const bool penalties = repetition || presence || frequency;
  const bool count = penalties && p.history;
  if (count && (!history || !starts)) return bad(BWPP_HIP_ERR_INVALID_ARG, "NULL history or starts");
  const uint64_t ex = p.dtype_x == BWPP_HIP_BF16 ? 2 : 4, ey = p.dtype_y == BWPP_HIP_BF16 ? 2 : 4;
  const bool in_place = x == y && ex == ey && (ldx == ldy || R == 1);
  const uint64_t ybytes = ((R - 1) * ldy + V) * ey;
  // Rows of y among other rows of one stride (columns of a wider buffer) meet none of them.
  bool alias = !in_place && (ex == ey ? bwpp_hip_blocks_overlap(y, R, V, ldy, x, R, V, ldx, ey)
                                      : bwpp_hip_blocks_overlap(y, 1, ybytes, 0, x, 1, ((R - 1) * ldx + V) * ex, 0, 1));
  const Span out = {y, ybytes};
  const Span small[8] = {{count ? history : nullptr, (uint64_t)p.history * 4},
                         {count ? starts : nullptr, (R + 1) * 4},
                         {count ? prompt : nullptr, R * 4},
                         {count ? repetition : nullptr, R * 4},
                         {count ? presence : nullptr, R * 4},
                         {count ? frequency : nullptr, R * 4},
                         {bias, (p.ld_bias ? (R - 1) * p.ld_bias + V : V) * 4},
                         {mask, (p.ld_mask ? (R - 1) * p.ld_mask + words : words) * 4}};
  for (const Span &s : small) alias = alias || meet(out, s);
  if (alias) return bad(BWPP_HIP_ERR_ALIAS, "y overlaps another operand");
  const BwppHipStatus s = bwpp_hip_enter(h);
  if (s != BWPP_HIP_OK) return s;
  BwppLogitArgs a = {};
  a.x = x;
  a.y = y;
  a.history = history;
  a.starts = starts;
  a.prompt = prompt;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias = bias;
  a.mask = mask;
  a.ldx = ldx;
  a.ldy = ldy;
  a.ld_bias = p.ld_bias;
  a.ld_mask = p.ld_mask;
  a.rows = p.rows;
  a.vocab = p.vocab;
  a.history_len = p.history;
  a.count = count ? 1u : 0u;
  // Wide chunks read the history less often; narrow ones fill the chip for few rows.
  a.chunk = 16384;
  while (a.chunk > 1024 && R * ((V + a.chunk - 1) / a.chunk) < 2ull * cus_of(h)) a.chunk /= 2;
  a.chunks = (uint32_t)((V + a.chunk - 1) / a.chunk);
  const uint32_t threads = a.chunk >= 8192 ? 1024u : 256u;
  return bwpp_hip_launch_cache(h, CK_RULES + (ex == 2 ? 2 : 0) + (ey == 2 ? 1 : 0), R * a.chunks, 1, threads, &a,
                               count ? a.chunk * 4 : 0);
}

/* Kernel argument blocks shared by the host runtime (g++) and the gfx950
 * kernels (hipcc).  Each kernel takes exactly one of these by value, so a
 * launch passes a single kernelParams entry to hipModuleLaunchKernel.
 * Plain C layout only: no HIP or C++ types. */
#ifndef BWPP_KARGS_H
#define BWPP_KARGS_H

#include <stdint.h>

/* Row-wise and column-wise reductions and their grads. */
typedef struct {
  const float *x;
  float *y; /* output rows (softmax/norm output, mask, dx) */
  const float *gamma;
  const float *beta;
  const float *dy; /* upstream grad: per line (reduce_max) or per element */
  const int32_t *idx_in;
  float *maxv;
  int32_t *argmax;
  float *part_v;    /* axis 0: [bands][cols] partial maxima ... */
  uint32_t *part_i; /* ... and their row indices */
  uint32_t rows;
  uint32_t cols;
  uint32_t ld;
  float eps;
  uint32_t bands;
} BwppRowArgs;

/* GEMM: C = op(A)·op(B) (+bias) (->SiLU); see gemm.hip. */
typedef struct {
  const void *a;
  const void *b;
  const void *bias; /* NULL: no bias even if the epilogue asks for one */
  void *c;
  uint32_t M;
  uint32_t N;
  uint32_t K;
  uint32_t lda;
  uint32_t ldb;
  uint32_t ldc;
  uint32_t epilogue; /* BWPP_HIP_EPILOGUE_* values */
  uint32_t tiles_m;  /* ceil(M / BM) */
  uint32_t tiles_n;  /* ceil(N / BN) */
  uint32_t group_m;  /* tile-order group height (in tiles) */
  uint32_t vec_ok;   /* 1: rows are 16-byte aligned (edge kernels only) */
  /* Split-K (fp32 full tiles): block b computes K range [s * kchunk, ..)
   * of tile b % tiles for s = b / tiles into part[s] ([M][N] raw sums);
   * bwpp_gemm_f32_splitk_reduce then applies the epilogue. */
  uint32_t ksplit;
  uint32_t kchunk;
  float *part;
  /* fp32 fusions after the epilogue (BWPP_HIP_FUSE_*): residual C += aux,
   * dual output c2 = SiLU(C), SiLU gradient C *= silu'(aux) */
  uint32_t fuse;
  uint32_t ldaux;
  const float *aux;
  float *c2;
  uint32_t ldc2;
} BwppGemmArgs;

/* Attention: O = softmax(scale * Q K^T [causal]) V per (batch, head). */
typedef struct {
  const void *q;
  const void *k;
  const void *v;
  void *o;
  uint32_t M; /* queries */
  uint32_t N; /* keys */
  uint32_t ldq, ldk, ldv, ldo;
  uint32_t heads;
  uint32_t q_tiles; /* ceil(M / queries per block) */
  uint64_t q_bs, q_hs, k_bs, k_hs, v_bs, v_hs, o_bs, o_hs;
  float scale_log2; /* scale * log2(e) (flash path); the plain scale (generic path) */
  uint32_t causal;
  uint32_t kdim; /* Q/K head dim (generic path) */
  uint32_t vdim; /* V/O head dim (generic path) */
  /* Forward: optional per-query log-sum-exp out ([B*H][M] fp32).
   * Backward: lse in, dout (O's strides), dq / dk / dv (Q / K / V strides),
   * dsum = rowsum(dout * o) scratch ([B*H][M] fp32). */
  float *lse;
  const void *dout;
  void *dq;
  void *dk;
  void *dv;
  float *dsum;
  float scale; /* the plain score scale (fp32 MFMA path, which gets scale * log2(e) in scale_log2) */
  uint32_t zigzag; /* fp32 MFMA causal kernels: tile order heavy ranks first, then the light ones
                      lightest first (a one-wave grid then pairs heavy with light on each CU) */
  /* Backward with a stored dS: dS^T written by the dK/dV pass and read by
   * the dQ pass, in blocks of 32 keys x 32 queries (bf16: DsBlk in
   * attention_bwd.hip, fp32: DsBlk32 in attention_f32.hip); ld_dst = the
   * query count rounded up to 128. */
  void *dst;
  uint32_t ld_dst;
  uint32_t items; /* persistent flash forward: (slice, query tile) items;
                     few queries: slices; generic path: rows per block */
  /* Few queries (decoding): the keys of a slice in ksplit ranges of kchunk;
   * with ksplit > 1, range s of slice b leaves its sums of p v
   * ([M][vdim]) at part_o + (b ksplit + s) M vdim and per query the pair
   * (exponent offset, sum of p) at part_ml + 2 (b ksplit + s) M. */
  uint32_t ksplit, kchunk;
  float *part_o, *part_ml;
} BwppAttnArgs;

/* Attention operand copies between the caller's strided bf16 layout
 * ([batch][head] slices of rows x cols, leading dimension ld) and
 * contiguous fp32 [batch * heads][rows][cols] (attention_f32.hip). */
typedef struct {
  const void *src;
  void *dst;
  uint64_t bs, hs;   /* batch / head strides of the bf16 side (elements) */
  uint32_t rows, cols, ld, heads;
  uint32_t slices;   /* batch * heads */
  uint32_t vec;      /* 1: bf16 rows are 16-byte aligned (8-element loads / stores) */
} BwppConvArgs;

/* Grad ops and elementwise glue (grad.hip). */
typedef struct {
  const float *a;   /* x, y or the left operand */
  const float *b;   /* dy or the right operand */
  const float *gamma;
  float *out;       /* dx or the result */
  float *out2;      /* dbeta (bwpp_col_partials_sum) */
  float *part_g;    /* [nblocks][cols] dgamma partials (rmsnorm_grad) */
  float *part_b;    /* [nblocks][cols] dbeta partials */
  uint64_t n;       /* element count (flat ops) */
  uint32_t rows;
  uint32_t cols;
  uint32_t ld;
  float eps;
  uint32_t op;      /* elementwise op */
  uint32_t bmode;   /* broadcast of b: 0 full, 1 row vector [cols], 2 column vector [rows], 3 scalar */
  uint32_t nparts;  /* partial rows to reduce */
  uint32_t vec;     /* 1: a, b, out are 16-byte aligned (flat ops); 16-byte
                       rows (elementwise) */
  uint32_t ldb;     /* elementwise, full broadcast: row stride of b */
  const float *acc; /* rmsnorm_grad: added to dx (row stride ld; may equal out) */
  const float *s_loss, *s_grad; /* mean_square: device scalars (NULL = 1) */
} BwppGradArgs;

/* Up to four strided copies in one launch (bwpp_copy_multi): segment s
 * copies rows row0[s] .. row0[s+1]-1 of the launch's row space. */
#define BWPP_COPY_MULTI_MAX 4
typedef struct {
  const float *src[BWPP_COPY_MULTI_MAX];
  float *dst[BWPP_COPY_MULTI_MAX];
  uint32_t ld_src[BWPP_COPY_MULTI_MAX], ld_dst[BWPP_COPY_MULTI_MAX], cols[BWPP_COPY_MULTI_MAX];
  uint32_t row0[BWPP_COPY_MULTI_MAX + 1];
  uint32_t n;   /* segments */
  uint32_t vec; /* 1: every segment has 16-byte rows (cols, strides, pointers) */
} BwppCopyArgs;

/* Rotary positions (rotary.h): rows of `dim` elements, one per (batch,
 * token, head), q's heads before k's. */
typedef struct {
  const void *q;
  const void *k;
  void *qo;
  void *ko;
  const int32_t *positions; /* [batch][pos_bs], or NULL: pos0 + token */
  uint64_t q_ts, q_hs, q_bs, k_ts, k_hs, k_bs;       /* token / head / batch strides (elements) */
  uint64_t qo_ts, qo_hs, qo_bs, ko_ts, ko_hs, ko_bs;
  uint64_t pos_bs;
  double log2_step; /* log2 of the ratio of two successive frequencies */
  double inv_factor;
  double turns;     /* context / (2 pi): turns of a frequency of 1 over the context */
  double low, inv_range; /* by parts: share kept = (turns f - low) inv_range in [0, 1] */
  float cos_scale, sin_scale; /* magnitude; the sine's sign is the direction */
  int32_t pos0;
  uint32_t tokens, batch;
  uint32_t q_heads, heads; /* heads = q's and k's */
  uint32_t dim, pairs;     /* pairs = rot_dim / 2 */
  uint32_t scaling;        /* BWPP_HIP_ROTARY_SCALE_* */
  uint32_t tile;           /* tokens per block */
  uint32_t hgroup;         /* heads per block (grid y), at most 256 */
  uint32_t copy;           /* bit 0: copy q's columns past 2 pairs, bit 1: k's */
  uint32_t tail_chunks;    /* chunks of those columns */
} BwppRotaryArgs;

/* The join of a branch with the residual stream and its gradient
 * (resnorm.h). */
typedef struct {
  const void *x, *o, *r;            /* stream in, branch, stream out (gradient: in) */
  const void *post, *gate, *pre;    /* weights, NULL = 1 */
  void *ro, *y;                     /* forward outputs */
  const void *dr, *dy;              /* upstream gradients, either NULL = 0 */
  void *dx, *dout, *dpost, *dgate, *dpre;
  float *part_pre, *part_post, *part_gate; /* [nparts][cols] sums (NULL: not asked for) */
  uint64_t ldx, ldo, ldy, ldg;
  uint32_t rows, cols;
  uint32_t gate_rows; /* rows per gate row (0: one gate row) */
  uint32_t post_norm;
  float eps, stream_scale, branch_scale;
  /* gradient: a group is the rows of one row of dgate.  split > 1: that many
   * blocks a group take its rows in turn, their gate sums go to part_gate; split = 1: workers (blocks, or waves of blocks where a wave
   * holds a row) take `span` rows each, whole groups.  nparts: blocks, one row
   * of partial sums each. */
  uint32_t workers, group, split, span, nparts;
} BwppResNormArgs;

/* Planes of bf16 terms of fp32 operands (gemm_bf16_k32.h): nibble t of *_planes
 * is the plane of the t-th of six products, planes are *_stride elements apart. */
typedef struct {
  uint32_t a_planes, b_planes;
  uint64_t a_stride, b_stride;
} BwppSplitTerms;

/* Cross entropy of hidden states against a vocabulary (xent.h).  Logits
 * z = scale op(W) x: g holds their product (M tokens, N of the columns n_base
 * .. of the vocabulary, K = dim). */
typedef struct {
  BwppGemmArgs g;
  const int32_t *target;
  const float *lse;   /* gradient */
  const float *dloss; /* gradient: NULL = 1 */
  uint32_t dloss_scalar;
  uint32_t n_base;
  uint32_t vocab;
  float scale;
  float *part; /* forward: [tiles][M] pairs (max, sum of exp(z - max)), ... */
  uint32_t part_base; /* ... of this launch from here */
  float *zt;   /* forward: [M] target logits */
  uint16_t *dl; /* gradient: dz scale, [M][ldl] bf16, ldl a multiple of 8 */
  uint32_t ldl;
  uint32_t rows_up; /* gradient: dl's rows, M and zeros behind (at most 31) */
  uint32_t rows_out, cols_out; /* rows product: what is stored of g.M x g.N */
  uint32_t accumulate; /* sums: add to what is there */
  float *raw;          /* sums: [ksplit][M][N] */
  BwppSplitTerms terms; /* fp32 operands in bf16 terms */
  uint64_t dl_stride;   /* gradient in terms: its three planes' distance; ... */
  uint32_t cols_up;     /* ... its columns, zeros behind N */
  float *rest;          /* gradient: [rows] what rounding left of the targets' dz scale */
  uint32_t rows;        /* rows product: tokens, and whether x is its A */
  uint32_t x_is_a;
} BwppXentArgs;

/* Its row kernels. */
typedef struct {
  const void *x;
  void *y;
  const float *src;      /* fp32 sums or logits */
  const int32_t *target;
  const float *dloss;
  const float *lse_in;
  float *part;
  float *zt;
  float *loss, *lse, *sums;
  uint64_t ldx, ldy, lds;
  uint32_t rows, cols, rows_up; /* rows_up: the copy's */
  uint32_t n_base, vocab;
  uint32_t nparts; /* partials a row, or planes of sums */
  uint32_t dloss_scalar;
  uint32_t lanes; /* join: rows a block; terms: threads a row; dx: tokens a block */
  uint64_t plane; /* terms: distance of the planes */
  const float *rest; /* bf16 sums: see BwppXentArgs, and W */
  const void *w;
  uint64_t ldw;
  float scale;
} BwppXentRowArgs;

/* A paged cache of keys and values and a ragged batch of new tokens
 * (kv_cache.h).  Strides in elements. */
typedef struct {
  void *k, *v;             /* pools of the same strides */
  const int32_t *table;    /* [batch][ld_table] page numbers */
  const int32_t *starts;   /* [batch + 1] first rows */
  const int32_t *held;     /* [batch] tokens in the cache before the new ones */
  uint64_t page_s, tok_s, head_s, ld_table;
  uint32_t pages, page_shift;
  uint32_t capacity;       /* slots of a sequence, below 2^31 */
  uint32_t batch, tokens, heads, dim;
} BwppCacheArgs;

/* New keys and values into their pages, q and k with rotary positions
 * (kv_append.h).  r: q, k, qo, their token and head strides, the rotation,
 * chunks; tile and hgroup as there, heads = q's + twice the cache's. */
typedef struct {
  BwppCacheArgs c;
  BwppRotaryArgs r;
  const void *v_in;
  uint64_t v_ts, v_hs;
} BwppCacheAppendArgs;

/* Accepted tokens moved together. */
typedef struct {
  BwppCacheArgs c;
  const int32_t *kept, *counts; /* [batch][ld_kept], [batch] */
  uint64_t ld_kept;
  uint32_t max_kept;
  uint32_t unit;   /* elements a chunk */
  uint32_t chunks; /* chunks a head's row */
} BwppCacheKeepArgs;

/* Attention of the new tokens over the cache (kv_attention.h).  Row r of a
 * sequence and key head is query head r % group of token r / group. */
typedef struct {
  BwppCacheArgs c;
  const void *q;
  void *o;
  float *lse;           /* [tokens][group * heads], or NULL */
  const uint32_t *mask; /* [tokens][mask_words], or NULL: causal */
  uint64_t q_ts, q_hs, o_ts, o_hs;
  uint32_t mask_words;
  uint32_t group;       /* query heads per key head */
  float scale_log2;     /* |scale| * log2(e) */
  uint32_t flip;        /* 1: the scale is negative */
  uint32_t blocks;      /* blocks that share the keys */
  double inv_blocks;    /* 1 / blocks */
  uint32_t whole_keys;  /* sequences up to here have whole items */
  uint32_t item_keys;   /* keys that an item costs by itself */
  uint64_t large_cost;  /* more is of more keys and values than the caches hold */
  float *part_o;        /* [2 blocks][rows of a tile][dim up to a multiple of 4] */
  float *part_ml;       /* [2 blocks][rows of a tile][2] */
} BwppCacheAttnArgs;

/* Rules for the next token on logits (logit_rules.h). */
typedef struct {
  const void *x;
  void *y;
  const int32_t *history, *starts, *prompt;
  const float *repetition, *presence, *frequency, *bias;
  const uint32_t *mask;
  uint64_t ldx, ldy, ld_bias, ld_mask;
  uint32_t rows, vocab;
  uint32_t chunk;  /* columns a block, a power of two, at most 16 a thread */
  uint32_t chunks; /* blocks a row */
  uint32_t history_len; /* elements of the history */
  uint32_t count;  /* 1: tokens of the history are counted */
} BwppLogitArgs;

#endif /* BWPP_KARGS_H */

/*
 * bwpp_hip.h -- C ABI of libbwpp_hip, the MI355X (gfx950) execution backend
 * for BW++'s hot ops.
 *
 * It replaces the reference's Metal operator seam
 * (runtime/metal/dispatch_stub.h:42-74, implemented in dispatch_stub.m) and
 * gives runtime/core's arena (runtime/core/arena.h:6-15) a device-memory
 * twin.  Kernels are hand-written gfx950 HIP, prebuilt into code objects
 * (*.hsaco) that bwpp_hip_create() loads with hipModuleLoad; every operator
 * launches with hipModuleLaunchKernel on the handle's stream.
 *
 * Conventions (kept from the reference):
 *  - the caller owns every buffer; pointers are device pointers unless a
 *    function says otherwise;
 *  - row-major with explicit leading dimensions (in elements); softmax and
 *    the norms run along the last axis;
 *  - a NULL gamma / beta / bias means 1 / 0 / 0 (dispatch_stub.m:103-110,
 *    215-234);
 *  - the params structs keep the reference's type names and leading fields,
 *    in the reference's order (dispatch_stub.h:9-40); fields added after them
 *    take their documented default when zero, so a reference-style
 *    initialiser `{M, N, K, lda, ldb, ldc}` keeps its meaning.
 * Differences:
 *  - every call returns a status instead of returning silently on bad
 *    arguments (dispatch_stub.m:66-79); a failed call launches nothing;
 *  - launches are asynchronous on the handle's stream; bwpp_hip_sync() waits
 *    (the reference waits inside every dispatch, dispatch_stub.m:139-140);
 *  - the function cache is filled once in bwpp_hip_create() and read-only
 *    afterwards (the reference's function-static PSO caches are not
 *    thread-safe, dispatch_stub.m:81), but a handle also holds its stream,
 *    its last-error text and the grad ops' workspace: use one handle per
 *    host thread, or serialise calls on a shared one.
 */
#ifndef BWPP_HIP_H
#define BWPP_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* 0 and 1 coincide with the reference's BwppStatus {BWPP_OK, BWPP_ERR}
 * (compiler/include/bwpp.h:8-11); the rest refine BWPP_ERR. */
typedef enum {
  BWPP_HIP_OK = 0,
  BWPP_HIP_ERR = 1,
  BWPP_HIP_ERR_INVALID_ARG = 2,   /* NULL pointer, bad size, ld < cols, ... */
  BWPP_HIP_ERR_HIP = 3,           /* a HIP runtime call failed */
  BWPP_HIP_ERR_NO_KERNEL = 4,     /* code object or kernel symbol missing */
  BWPP_HIP_ERR_ALIAS = 5,         /* GEMM/attention output overlaps an input */
  BWPP_HIP_ERR_OUT_OF_MEMORY = 6, /* device allocation or arena exhausted */
  BWPP_HIP_ERR_UNSUPPORTED = 7,   /* valid request this build does not run */
  BWPP_HIP_ERR_NO_DEVICE = 8      /* no usable HIP device */
} BwppHipStatus;

typedef enum { BWPP_HIP_F32 = 0, BWPP_HIP_BF16 = 1 } BwppHipDType;

/* Same values as BwppTileEpilogue (compiler/include/tile_ir.h:35-40). */
typedef enum {
  BWPP_HIP_EPILOGUE_NONE = 0,
  BWPP_HIP_EPILOGUE_ADD = 1,
  BWPP_HIP_EPILOGUE_SILU = 2,
  BWPP_HIP_EPILOGUE_ADD_SILU = 3
} BwppHipEpilogue;

/* dispatch_stub.h:9-16 + extensions.
 * C = op(A)·op(B) (+bias[col]) (→SiLU).  A is [M x K] (trans_a: stored
 * [K x M]), B is [K x N] (trans_b: stored [N x K]); lda/ldb/ldc are the row
 * strides of the stored matrices.  dtype F32: fp32 in/out on FP32 MFMA;
 * BF16: bf16 A, B, bias and C with fp32 accumulation and epilogue, C rounded
 * to nearest even.  bias is read only when the epilogue includes ADD. */
typedef struct {
  uint32_t M;
  uint32_t N;
  uint32_t K;
  uint32_t lda;
  uint32_t ldb;
  uint32_t ldc;
  uint32_t dtype;    /* BwppHipDType, 0 = F32 */
  uint32_t epilogue; /* BwppHipEpilogue, 0 = none */
  uint32_t trans_a;  /* 0 = A row-major [M x K] */
  uint32_t trans_b;  /* 0 = B row-major [K x N] */
} BwppMatmulParams;

/* dispatch_stub.h:18-22.  ld is the row stride of x and y (0 = cols). */
typedef struct {
  uint32_t rows;
  uint32_t cols;
  uint32_t ld;
} BwppSoftmaxParams;

/* dispatch_stub.h:24-29; also used by LayerNorm and the norm grads.
 * ld is the row stride of x, y and dy (0 = cols). */
typedef struct {
  uint32_t rows;
  uint32_t cols;
  uint32_t ld;
  float eps;
} BwppRmsnormParams;

/* dispatch_stub.h:31-40 + extensions.  One (batch, head) slice is the
 * reference's single-head problem: Q [M x K], K [N x K], V [N x D],
 * O [M x D] with row strides ldq/ldk/ldv/ldo; slices are placed by the
 * batch/head strides (elements).  O = softmax(scale * Q·K^T [masked]) · V.
 * causal masks keys n > m + (N - M) (bottom-right aligned; rows that see no
 * key produce zeros).  dtype BF16: bf16 Q/K/V/O, fp32 softmax and
 * accumulation; F32: fp32 throughout. */
typedef struct {
  uint32_t M;
  uint32_t N;
  uint32_t K;
  uint32_t D;
  uint32_t ldq;
  uint32_t ldk;
  uint32_t ldv;
  uint32_t ldo;
  uint32_t batch; /* 0 = 1 */
  uint32_t heads; /* 0 = 1 */
  uint64_t q_batch_stride, q_head_stride;
  uint64_t k_batch_stride, k_head_stride;
  uint64_t v_batch_stride, v_head_stride;
  uint64_t o_batch_stride, o_head_stride;
  float scale;     /* 0 = 1.0: the reference applies no scale */
  uint32_t causal; /* 0 = unmasked, as the reference */
  uint32_t dtype;  /* BwppHipDType, 0 = F32 */
} BwppAttentionParams;

/* reduce_max family.  axis follows bwpp_cpu_ref.c:156,172: axis == 0 reduces
 * over rows (one result per column), any other value reduces along each row
 * (one result per row). */
typedef struct {
  uint32_t rows;
  uint32_t cols;
  uint32_t ld; /* row stride of x / mask / dx; 0 = cols */
  int32_t axis;
} BwppReduceParams;

/* Elementwise glue of the autodiff graph (graph_ir.c:697-770, 1457-1470,
 * 1585-1654): out = a (op) b with b broadcast as selected; op COPY writes
 * the broadcast b and op SILU its SiLU b / (1 + expf(-b)) (graph op
 * BWPP_GOP_SILU, bwpp_cpu_ref.c:4-6; a unused for both).  rows x cols with
 * leading dimension ld (0 = cols) for a, out and a full b. */
typedef enum {
  BWPP_HIP_OP_ADD = 0,
  BWPP_HIP_OP_SUB = 1,
  BWPP_HIP_OP_MUL = 2,
  BWPP_HIP_OP_DIV = 3,
  BWPP_HIP_OP_COPY = 4,
  BWPP_HIP_OP_SILU = 5
} BwppHipElementwiseOp;
typedef enum {
  BWPP_HIP_BCAST_FULL = 0,   /* b is rows x cols */
  BWPP_HIP_BCAST_ROW = 1,    /* b[cols], repeated for every row */
  BWPP_HIP_BCAST_COL = 2,    /* b[rows], repeated along each row */
  BWPP_HIP_BCAST_SCALAR = 3  /* b[0] */
} BwppHipBroadcast;
typedef struct {
  uint32_t rows;
  uint32_t cols;
  uint32_t ld;
  uint32_t op;    /* BwppHipElementwiseOp */
  uint32_t bmode; /* BwppHipBroadcast */
} BwppElementwiseParams;

/* Rotary positions of one attention call's q and k (no reference
 * counterpart; strides named as BwppAttentionParams names them, the outputs'
 * with an o).  Row (b, t, h) of q is at b * q_batch_stride + t * ldq + h *
 * q_head_stride (elements), `dim` long; zero strides mean contiguous [batch,
 * heads, tokens, dim].  The first rot_dim columns are n/2 = rot_dim/2 pairs:
 * (i, i + n/2) (HALF) or (2i, 2i + 1) (INTERLEAVED); pair i of a token at
 * position p turns by p * f_i, f_i = base^(-2i/n), and is multiplied by
 * `magnitude`; the other columns are copied.  For contexts longer than the
 * one trained on: LINEAR divides every f_i by `factor`; BY_PARTS divides by
 * parts, f_i (c + (1 - c) / factor) with c = (r - low_turns) / (high_turns -
 * low_turns) cut to 0..1 and r = context * f_i / (2 pi), the turns of the pair
 * over `context` positions: fast pairs keep their frequency. */
typedef enum { BWPP_HIP_ROTARY_HALF = 0, BWPP_HIP_ROTARY_INTERLEAVED = 1 } BwppHipRotaryLayout;
typedef enum {
  BWPP_HIP_ROTARY_SCALE_NONE = 0,
  BWPP_HIP_ROTARY_SCALE_LINEAR = 1,
  BWPP_HIP_ROTARY_SCALE_BY_PARTS = 2
} BwppHipRotaryScaling;
typedef struct {
  uint32_t tokens;
  uint32_t q_heads;
  uint32_t k_heads;
  uint32_t dim;
  uint32_t batch;   /* 0 = 1 */
  uint32_t rot_dim; /* even, at most dim and 4096; 0 = dim.  dim and tokens: at most
                       2^31, heads of q and k 2^24 */
  uint32_t layout;  /* BwppHipRotaryLayout */
  uint32_t dtype;   /* BwppHipDType, 0 = F32 */
  uint32_t ldq, ldk, ldqo, ldko; /* token strides; 0 = dim */
  uint64_t q_batch_stride, q_head_stride;
  uint64_t k_batch_stride, k_head_stride;
  uint64_t qo_batch_stride, qo_head_stride;
  uint64_t ko_batch_stride, ko_head_stride;
  uint64_t pos_batch_stride; /* positions of a batch; 0 = the same for all */
  int32_t pos_offset;        /* without positions: token t is at pos_offset + t */
  uint32_t scaling;          /* BwppHipRotaryScaling */
  float base;                /* 0 = 10000 */
  float factor;              /* 0 = 1 */
  float low_turns, high_turns;
  uint32_t context;
  float magnitude;           /* 0 = 1 */
} BwppRotaryParams;

/* The join of a block's branch o with the residual stream x, and the norms
 * around it (no reference counterpart).  With v' = v / sqrt(mean(v^2) + eps)
 * along the rows:
 *   u = post_gamma o'   (post_norm = 0: u = o)
 *   r = stream_scale x + branch_scale gate u
 *   y = pre_gamma r'    (the next block's input)
 * gate row i / gate_rows applies to row i (0: one gate row for all; 1: a gate
 * of o's shape).  x, r and their gradients have row stride ldx, o and its
 * gradient ldo, y and its gradient ldy, gate rows ldg. */
typedef struct {
  uint32_t rows;
  uint32_t cols; /* fewer than 2^31, for weight and gate gradients at most 2^28 - 64 */
  uint32_t ldx, ldo, ldy, ldg; /* 0 = cols */
  uint32_t post_norm;
  uint32_t gate_rows;
  float eps;
  float stream_scale; /* 0 = 1 */
  float branch_scale; /* 0 = 1 */
  uint32_t dtype;     /* BwppHipDType of every operand, 0 = F32 */
} BwppResidualNormParams;

/* Cross entropy of hidden states x [rows x dim] against a vocabulary, logits
 * z = scale x W, W [dim x vocab] (trans_w: stored [vocab x dim]), without the
 * logits in memory (no reference counterpart; its compiler has no loss). */
typedef struct {
  uint32_t rows; /* tokens, fewer than 2^27 */
  uint32_t vocab;
  uint32_t dim;
  uint32_t ldx, ldw;   /* row strides of the stored matrices; 0 = contiguous */
  uint32_t lddx, lddw; /* of the gradients (dW is stored as W is) */
  uint32_t trans_w;
  uint32_t dtype;        /* BwppHipDType of x, W and their gradients, 0 = F32 */
  uint32_t dloss_scalar; /* the upstream gradient is one value for all rows */
  float scale;           /* 0 = 1 */
} BwppLinearXentParams;

/* A cache of keys and values in pages, and a ragged batch of new tokens over it
 * (no reference counterpart).  The pools of keys and values have `pages` pages of
 * page_tokens tokens and the same strides (elements); zero strides mean contiguous
 * [pages][heads][page_tokens][dim] (token_stride 0 = dim, head_stride 0 =
 * page_tokens token_stride, page_stride 0 = heads head_stride).  In device memory,
 * so that a recorded launch follows them:
 *   table   int32 [batch][max_pages], row stride ld_table: page numbers
 *   starts  int32 [batch + 1], not descending: new tokens of sequence s are rows
 *           starts[s] .. starts[s + 1] - 1 of the operands' `tokens` rows; rows
 *           before the first and behind the last sequence are left alone
 *   held    int32 [batch]: tokens that the cache holds before the new ones, which
 *           take the slots behind them
 * Slot p of a sequence lies in page table[s][p / page_tokens].  Starts are cut to
 * the operands, lengths below zero are none; a slot past the table (or from 2^31 - 1
 * on), or whose page number is outside 0 .. pages - 1 (-1: no page), does not exist:
 * nothing is written there and no query sees it. */
typedef struct {
  uint32_t pages;
  uint32_t page_tokens; /* a power of two */
  uint32_t heads;       /* key (and value) heads */
  uint32_t dim;         /* of a key and of a value */
  uint32_t batch;       /* sequences, at most 2^24 */
  uint32_t max_pages;   /* columns of the table */
  uint32_t ld_table;    /* 0 = max_pages */
  uint32_t tokens;      /* rows of the new tokens' operands */
  uint32_t q_heads;     /* a multiple of heads; tokens q_heads below 2^31 */
  uint32_t dtype;       /* BwppHipDType of every operand that is not int32 or lse */
  uint64_t page_stride, token_stride, head_stride;
} BwppCacheParams;

/* Rows of the new tokens: zero strides mean contiguous [tokens][heads][dim]
 * (heads: v's are k's).  The rotation is BwppRotaryParams', fields as there. */
typedef struct {
  BwppCacheParams cache;
  uint32_t ldq, ldk, ldv, ldqo; /* token strides; 0 = heads * dim */
  uint64_t q_head_stride, k_head_stride, v_head_stride, qo_head_stride; /* 0 = dim */
  uint32_t no_rotation; /* 1: q and k as they are */
  uint32_t rot_dim;     /* 0 = dim */
  uint32_t layout;
  uint32_t scaling;
  float base;
  float factor;
  float low_turns, high_turns;
  uint32_t context;
  float magnitude;
} BwppCacheAppendParams;

typedef struct {
  BwppCacheParams cache; /* dim at most 256 */
  uint32_t ldq, ldo;     /* token strides; 0 = q_heads * dim */
  uint64_t q_head_stride, o_head_stride; /* 0 = dim */
  uint32_t mask_words;   /* 32-bit words a row of the mask */
  float scale;           /* 0 = 1 */
} BwppCacheAttentionParams;

typedef struct {
  BwppCacheParams cache; /* tokens and q_heads are not read */
  uint32_t max_kept;     /* columns of kept */
  uint32_t ld_kept;      /* 0 = max_kept */
} BwppCacheKeepParams;

/* Rules for the next token on rows of logits (no reference counterpart). */
typedef struct {
  uint32_t rows;
  uint32_t vocab;
  uint32_t ldx, ldy;  /* 0 = vocab */
  uint32_t dtype_x, dtype_y; /* BwppHipDType, 0 = F32 */
  uint32_t history;   /* tokens of the history, all rows together */
  uint32_t ld_bias;   /* 0: one row for all */
  uint32_t ld_mask;   /* 32-bit words; 0: one row for all */
} BwppLogitRulesParams;

typedef struct BwppHip BwppHip;

/* ---- handle ---- */

/* Selects `device`, loads every code object from code_object_dir (NULL: the
 * directory holding libbwpp_hip.so) and resolves every kernel.  Fails with
 * NO_DEVICE / NO_KERNEL / HIP rather than returning a half-built handle.
 * Replaces the per-op PSO cache (dispatch_stub.m:6-56). */
BwppHipStatus bwpp_hip_create(BwppHip **out, int device,
                              const char *code_object_dir);
void bwpp_hip_destroy(BwppHip *h);
/* Stream for subsequent launches (a hipStream_t); NULL = the null stream.
 * The handle's workspace (split-K partials of fp32 products, attention-
 * backward row sums, column partials, pieces of a cross entropy's logits) is ordered on the handle's stream: when
 * the stream changes, the new stream first waits for the work queued on the
 * old one.
 *
 * Besides the workspace a handle has one scratch of 64 MiB, allocated by the
 * first call that splits its work through it (bf16 and ragged fp32 products
 * over K, attention with at most 32 queries over the keys, reduce_max and its
 * mask and gradient over rows) and kept until bwpp_hip_destroy.  Calls without
 * it take other kernels or no split, with the same results up to the order of
 * sums: where it cannot be allocated, and in a graph that the caller records,
 * which may run beside this handle's other work (plans recorded by
 * bwpp_hip_plan_capture do use it).  A use of it on another stream waits for
 * the last one; changing the stream while the old one is being recorded
 * leaves no way to wait, and the handle then goes on without the scratch.
 * A graph that the caller records addresses the workspace as it then is: run
 * the calls once before, and record again after a call that needs more.  Such
 * graphs, and the handle's other work, write the same workspace: replay them
 * one after another (on one stream, or with events between).  The workspace
 * grows to the largest call's and is freed by bwpp_hip_destroy. */
BwppHipStatus bwpp_hip_set_stream(BwppHip *h, void *hip_stream);
void *bwpp_hip_get_stream(const BwppHip *h);
/* Waits for all work on the handle's stream. */
BwppHipStatus bwpp_hip_sync(BwppHip *h);
/* Text of the last failure on this handle ("" if none). */
const char *bwpp_hip_last_error(const BwppHip *h);
const char *bwpp_hip_status_string(BwppHipStatus s);
/* Number of compute units of the handle's device (for launch heuristics). */
int bwpp_hip_device_cus(const BwppHip *h);
/* Symbol of the last kernel this handle launched ("" if none): which
 * variant a dispatch chose.  No reference counterpart (diagnostics). */
const char *bwpp_hip_last_kernel(const BwppHip *h);
/* Symbol of the launch `back` launches before the last (0 = the last, at
 * most 3; "" if none): the kernels of a dispatch that launches several,
 * e.g. a split-K GEMM and its reduce.  No reference counterpart
 * (diagnostics). */
const char *bwpp_hip_recent_kernel(const BwppHip *h, int back);

/* ---- device memory ---- */

/* Device twin of runtime/core/arena.h:6-15 / arena.c:4-38: one hipMalloc of
 * `capacity` bytes, bump allocation with power-of-two alignment, NULL on
 * exhaustion, reset rewinds, destroy frees. */
typedef struct {
  unsigned char *buffer; /* device address */
  size_t capacity;
  size_t offset;
  int device;
} BwppHipArena;

BwppHipStatus bwpp_hip_arena_init(BwppHip *h, BwppHipArena *arena,
                                  size_t capacity);
void bwpp_hip_arena_reset(BwppHipArena *arena);
void *bwpp_hip_arena_alloc(BwppHipArena *arena, size_t size, size_t align);
void bwpp_hip_arena_destroy(BwppHipArena *arena);

/* ---- tensor metadata (device twin of runtime/core/tensor.h) ---- */

/* The three dtype numberings met on the path:
 *   runtime/core BwppDType (runtime/core/tensor.h:7-11): F16 0, BF16 1, F32 2
 *   compiler BwppDType (compiler/include/graph_ir.h:18-23):
 *                                            UNKNOWN 0, F16 1, BF16 2, F32 3
 *   BwppHipDType (above):                    F32 0, BF16 1
 * BwppHipTensor carries runtime/core's numbering, as BwppTensor does; the
 * mappers below convert between them and return -1 for a dtype with no
 * counterpart (compiler UNKNOWN; F16, for which this build has no
 * kernels). */
typedef enum {
  BWPP_HIP_CORE_F16 = 0,
  BWPP_HIP_CORE_BF16 = 1,
  BWPP_HIP_CORE_F32 = 2
} BwppHipCoreDType;
typedef enum {
  BWPP_HIP_LAYOUT_ROW_MAJOR = 0, /* runtime/core/tensor.h:13-16 */
  BWPP_HIP_LAYOUT_COL_MAJOR = 1
} BwppHipLayout;

/* runtime/core/tensor.h:18-25 with a device buffer: same fields, order and
 * widths (the enums are int-sized), so a BwppTensor that describes device
 * memory has this layout.  stride[i] is in elements; a contiguous
 * row-major tensor has stride[rank-1] = 1.  COL_MAJOR marks a rank-2
 * tensor stored transposed (stride[0] = 1, stride[1] = leading dim). */
typedef struct {
  int32_t dtype;  /* BwppHipCoreDType */
  int32_t layout; /* BwppHipLayout */
  uint32_t rank;  /* 1..4 */
  uint64_t shape[4];
  uint64_t stride[4];
  void *buffer;   /* device address */
} BwppHipTensor;

int32_t bwpp_hip_dtype_from_core(int32_t core_dtype);   /* -> BwppHipDType */
int32_t bwpp_hip_dtype_from_graph(int32_t graph_dtype); /* -> BwppHipDType */
int32_t bwpp_hip_dtype_to_core(int32_t hip_dtype);      /* -> runtime/core */
int32_t bwpp_hip_dtype_to_graph(int32_t hip_dtype);     /* -> compiler */
/* Bytes per element of a runtime/core dtype (0 if unknown). */
size_t bwpp_hip_core_dtype_size(int32_t core_dtype);

/* Describes `buffer` as a contiguous tensor of `rank` dims in the given
 * layout (COL_MAJOR needs rank 2).  buffer may be NULL (shape only). */
BwppHipStatus bwpp_hip_tensor_init(BwppHipTensor *t, int32_t core_dtype,
                                   int32_t layout, uint32_t rank,
                                   const uint64_t *shape, void *buffer);
/* Bytes spanned by the tensor's elements (its strides included). */
size_t bwpp_hip_tensor_bytes(const BwppHipTensor *t);
/* bwpp_hip_tensor_init over memory taken from a device arena (256-byte
 * aligned); OUT_OF_MEMORY when the arena is exhausted. */
BwppHipStatus bwpp_hip_tensor_alloc(BwppHipArena *arena, BwppHipTensor *t,
                                    int32_t core_dtype, int32_t layout,
                                    uint32_t rank, const uint64_t *shape);
/* The [rows x cols] matrix with row stride ld (elements) that a row-major
 * tensor is to the row operators: cols = last dim, rows = product of the
 * others, which must be stacked at one stride.  UNSUPPORTED otherwise. */
BwppHipStatus bwpp_hip_tensor_matrix(const BwppHipTensor *t, uint32_t *rows,
                                     uint32_t *cols, uint32_t *ld);

/* Tensor-level forms of the operators below: parameters come from the
 * metadata (dtype, shape, strides, layout).  C = A·B (+bias) (→SiLU) with A
 * [M,K], B [K,N], C [M,N] rank 2 (a COL_MAJOR A or B runs transposed);
 * softmax / rmsnorm / layernorm along the last dim of any rank; attention
 * over rank-4 [batch, heads, seq, dim] q, k, v, o (slice strides from the
 * tensors).  dtypes must agree (f32, or bf16 for matmul / attention). */
BwppHipStatus bwpp_hip_tensor_matmul(BwppHip *h, const BwppHipTensor *a,
                                     const BwppHipTensor *b,
                                     const BwppHipTensor *bias,
                                     BwppHipTensor *c, uint32_t epilogue);
BwppHipStatus bwpp_hip_tensor_softmax(BwppHip *h, const BwppHipTensor *x,
                                      BwppHipTensor *y);
BwppHipStatus bwpp_hip_tensor_rmsnorm(BwppHip *h, const BwppHipTensor *x,
                                      const BwppHipTensor *gamma,
                                      const BwppHipTensor *beta,
                                      BwppHipTensor *y, float eps);
BwppHipStatus bwpp_hip_tensor_layernorm(BwppHip *h, const BwppHipTensor *x,
                                        const BwppHipTensor *gamma,
                                        const BwppHipTensor *beta,
                                        BwppHipTensor *y, float eps);
BwppHipStatus bwpp_hip_tensor_attention(BwppHip *h, const BwppHipTensor *q,
                                        const BwppHipTensor *k,
                                        const BwppHipTensor *v,
                                        BwppHipTensor *o, float scale,
                                        uint32_t causal);

/* Stream-ordered copies, complete on return. */
BwppHipStatus bwpp_hip_copy_to_device(BwppHip *h, void *dst, const void *src,
                                      size_t bytes);
BwppHipStatus bwpp_hip_copy_to_host(BwppHip *h, void *dst, const void *src,
                                    size_t bytes);

/* ---- operators (device pointers; asynchronous on the handle's stream) ---- */

/* bwpp_metal_dispatch_matmul (dispatch_stub.h:42-49); CPU twin
 * bwpp_cpu_matmul_f32 (bwpp_cpu_ref.c:8-35).  C must not overlap A, B or
 * bias (ALIAS). */
BwppHipStatus bwpp_hip_dispatch_matmul(BwppHip *h, const void *a,
                                       const void *b, void *c,
                                       const void *bias,
                                       BwppMatmulParams params);

/* Matmul with a fused elementwise tail (no reference counterpart: the
 * HIP lowering's fusions of the graph's add / silu / silu_grad nodes into
 * the GEMM that feeds them).  fp32 only (dtype F32, else UNSUPPORTED).
 * After the params' bias / SiLU epilogue, with Y = that result:
 *   RESIDUAL   C = Y + aux        (aux [M x N], row stride ld_aux; aux may
 *                                  be C itself, with ld_aux = ldc)
 *   DUAL_SILU  C = Y, c2 = SiLU(Y) (c2 [M x N], row stride ld_c2; the
 *                                  params' epilogue may not include SiLU)
 *   SILU_GRAD  C = Y * s (1 + x (1 - s)), x = aux, s = 1 / (1 + e^-x)
 *                                 (the graph's silu_grad with Y as dY;
 *                                  epilogue must be NONE)
 * NONE is bwpp_hip_dispatch_matmul. */
typedef enum {
  BWPP_HIP_FUSE_NONE = 0,
  BWPP_HIP_FUSE_RESIDUAL = 1,
  BWPP_HIP_FUSE_DUAL_SILU = 2,
  BWPP_HIP_FUSE_SILU_GRAD = 3
} BwppHipFusion;

typedef struct {
  uint32_t kind;   /* BwppHipFusion */
  uint32_t ld_aux; /* 0 = N */
  uint32_t ld_c2;  /* 0 = N */
} BwppHipFusionParams;

BwppHipStatus bwpp_hip_dispatch_matmul_fused(BwppHip *h, const void *a,
                                             const void *b, void *c,
                                             const void *bias,
                                             const float *aux, float *c2,
                                             BwppMatmulParams params,
                                             BwppHipFusionParams fusion);

/* bwpp_metal_dispatch_softmax (dispatch_stub.h:51-56); CPU twin
 * bwpp_cpu_softmax_f32 (bwpp_cpu_ref.c:37-61).  y may equal x. */
BwppHipStatus bwpp_hip_dispatch_softmax(BwppHip *h, const float *x, float *y,
                                        BwppSoftmaxParams params);

/* bwpp_metal_dispatch_rmsnorm (dispatch_stub.h:58-65); CPU twin
 * bwpp_cpu_rmsnorm_f32 (bwpp_cpu_ref.c:63-90).  y may equal x. */
BwppHipStatus bwpp_hip_dispatch_rmsnorm(BwppHip *h, const float *x,
                                        const float *gamma, const float *beta,
                                        float *y, BwppRmsnormParams params);

/* LayerNorm: no reference kernel (ROADMAP.md:14); same argument order as
 * rmsnorm.  y = (x-mean)/sqrt(var+eps)*gamma+beta, population variance. */
BwppHipStatus bwpp_hip_dispatch_layernorm(BwppHip *h, const float *x,
                                          const float *gamma,
                                          const float *beta, float *y,
                                          BwppRmsnormParams params);

/* bwpp_metal_dispatch_attention (dispatch_stub.h:67-74); CPU twin
 * bwpp_cpu_attention_f32 (bwpp_cpu_ref.c:92-144).  O must not overlap Q, K
 * or V (ALIAS). */
BwppHipStatus bwpp_hip_dispatch_attention(BwppHip *h, const void *q,
                                          const void *k, const void *v,
                                          void *o, BwppAttentionParams params);

/* Forward attention that also writes lse[(b*H + h)*M + m], the natural-log
 * log-sum-exp of query m's scaled, masked scores (-inf when it sees no key),
 * for the backward below.  No reference counterpart (the reference
 * differentiates attention through its decomposed graph ops,
 * graph_ir.c:1722-1733, 1529-1583).  The same kernels as the plain forward
 * run: bf16 with K = D = 32, 64, 96 or 128, 16-byte rows (pointers, leading
 * dims and slice strides in multiples of 8 elements) and a positive scale
 * takes the bf16 matrix-core kernels; fp32 with K = D = 64 or 128 and 16-byte
 * rows the fp32 ones; both have kernels of their own for at most 32 queries
 * (K = D = 64 or 128); anything else takes the generic kernel.  A key that a
 * query does not see has weight 0.  With more than 32 queries the fp32
 * matrix-core kernel and the bf16 one for K = D = 128 multiply V by that
 * weight, so there an infinite or NaN V at a hidden key can turn a query of
 * the same tile into NaN; the other kernels leave hidden keys out. */
BwppHipStatus bwpp_hip_dispatch_attention_lse(BwppHip *h, const void *q,
                                              const void *k, const void *v,
                                              void *o, float *lse,
                                              BwppAttentionParams params);

/* Attention backward: dq, dk, dv of O = softmax(scale Q K^T [causal]) V
 * for the upstream gradient dout, from q, k, v, o and the forward's lse.
 * dout / dq / dk / dv use the strides of o / q / k / v.  Outputs must not
 * overlap inputs or each other.  Uses the handle's workspace for
 * rowsum(dout * o) and, for bf16 with K = D = 128 and for the fp32
 * matrix-core shapes, for dS (2 or 4 bytes x batch * heads *
 * ceil(N / 32) * 32 * ceil(M / 128) * 128, up to BWPP_ATTN_BWD_DS_MB MiB,
 * default 8192; beyond that, with 0, or when the device cannot allocate
 * it, S and dP are recomputed instead, with the same results).  Replaces the decomposed path of
 * graph_ir.c:1722-1733 (softmax_grad over materialised probabilities). */
BwppHipStatus bwpp_hip_dispatch_attention_grad(BwppHip *h, const void *q,
                                               const void *k, const void *v,
                                               const void *o, const void *dout,
                                               const float *lse, void *dq,
                                               void *dk, void *dv,
                                               BwppAttentionParams params);

/* bwpp_hip_dispatch_attention_grad that allocates nothing: no reference
 * counterpart; for callers that cannot call hipMalloc (code under HIP graph
 * capture, tight serving loops, harnesses that forbid allocation).  The
 * per-query row sums rowsum(dout * o) live in a device-resident scratch
 * array of the library (8 MiB per GPU, held until the process ends)
 * instead of the handle's workspace, so batch * heads * M may be at most
 * 2,097,151 query rows (UNSUPPORTED beyond, nothing launched).  bf16 rows
 * that are not 16-byte aligned (which need fp32 copies in the workspace)
 * are UNSUPPORTED too.  Every call on one GPU shares that GPU's scratch:
 * calls that overlap on one GPU (several streams, handles or threads) race
 * on it; calls ordered on one stream do not.  Results are bit-identical to
 * bwpp_hip_dispatch_attention_grad's (but for the sign of a zero that is
 * an all-zero sum: this entry recomputes S and dP in the dQ pass rather
 * than storing dS). */
BwppHipStatus bwpp_hip_dispatch_attention_grad_noalloc(
    BwppHip *h, const void *q, const void *k, const void *v, const void *o,
    const void *dout, const float *lse, void *dq, void *dk, void *dv,
    BwppAttentionParams params);

/* reduce_max forward (graph op BWPP_GOP_REDUCE_MAX, graph_ir.h:48; no
 * reference kernel): maxv as the reference's fold, argmax = lowest index
 * holding it (-1 if none).  Either output may be NULL, not both. */
BwppHipStatus bwpp_hip_dispatch_reduce_max(BwppHip *h, const float *x,
                                           float *maxv, int32_t *argmax,
                                           BwppReduceParams params);

/* bwpp_cpu_reduce_max_mask_f32 (bwpp_cpu_ref.c:146-190): 1.0 at every
 * element equal to its line's maximum, else 0.0. */
BwppHipStatus bwpp_hip_dispatch_reduce_max_mask(BwppHip *h, const float *x,
                                                float *mask,
                                                BwppReduceParams params);

/* bwpp_cpu_reduce_max_grad_f32 (bwpp_cpu_ref.c:192-219): dx = mask * dy,
 * dy broadcast along the reduced axis. */
BwppHipStatus bwpp_hip_dispatch_reduce_max_grad(BwppHip *h, const float *mask,
                                                const float *dy, float *dx,
                                                BwppReduceParams params);

/* reduce_max grad routed one-hot to the lowest-index maximum: pass x (the
 * argmax is recomputed in the same pass) or argmax (saved indices), not
 * both NULL; dx is fully written. */
BwppHipStatus bwpp_hip_dispatch_reduce_max_grad_argmax(
    BwppHip *h, const float *x, const int32_t *argmax, const float *dy,
    float *dx, BwppReduceParams params);

/* ---- autodiff grad ops (graph_ir.c:1485-1839 emits them; the reference
 * has no numeric kernels, the closed forms are in oracle/bwpp_oracle.h) ---- */

/* BWPP_GOP_SILU_GRAD (graph_ir.c:1709-1720), n contiguous elements:
 * s = 1/(1+e^-x); dx = dy * s * (1 + x (1 - s)). */
BwppHipStatus bwpp_hip_dispatch_silu_grad(BwppHip *h, const float *x, const float *dy, float *dx,
                                          uint64_t n);

/* BWPP_GOP_SOFTMAX_GRAD (graph_ir.c:1722-1733), along rows:
 * dx = y * (dy - sum_c dy*y). */
BwppHipStatus bwpp_hip_dispatch_softmax_grad(BwppHip *h, const float *y, const float *dy, float *dx,
                                             BwppSoftmaxParams params);

/* BWPP_GOP_RMSNORM_GRAD (graph_ir.c:1735-1789): dx for every row, and the
 * column sums dgamma = sum_r dy * xhat, dbeta = sum_r dy when those
 * pointers are non-NULL (needs cols <= 8192).  gamma NULL means 1. */
BwppHipStatus bwpp_hip_dispatch_rmsnorm_grad(BwppHip *h, const float *x, const float *gamma,
                                             const float *dy, float *dx, float *dgamma,
                                             float *dbeta, BwppRmsnormParams params);

/* bwpp_hip_dispatch_rmsnorm_grad with dx = acc + the gradient: the
 * autodiff graph's add of the residual branch's gradient
 * (graph_ir.c:1529-1545, ADD of the two gradient contributions to x) folded
 * into the same pass, with one fp32 rounding like the separate add.  acc has
 * dx's layout (row stride params.ld) and may be dx itself; NULL acc is
 * bwpp_hip_dispatch_rmsnorm_grad. */
BwppHipStatus bwpp_hip_dispatch_rmsnorm_grad_acc(BwppHip *h, const float *x, const float *gamma,
                                                 const float *dy, const float *acc, float *dx,
                                                 float *dgamma, float *dbeta,
                                                 BwppRmsnormParams params);

/* Mean-square training loss and its gradient, the loss the HIP target's
 * `--train mean_square` appends (no reference counterpart: the reference
 * compiler has no loss; the C5 configuration names loss = mean(out^2)):
 * loss[0] = loss_scale * sum of x^2 over rows x cols, and dx = grad_scale * x
 * when dx is non-NULL (dx may be x).  The scales are device scalars (NULL
 * = 1), e.g. 1/n and 2/n.  One pass over x plus a one-block finish; the sum
 * is taken in a fixed order (deterministic for a given device).  Either
 * output may be NULL, not both. */
typedef struct {
  uint32_t rows;
  uint32_t cols;
  uint32_t ld; /* row stride of x and dx; 0 = cols */
} BwppMeanSquareParams;

BwppHipStatus bwpp_hip_dispatch_mean_square(BwppHip *h, const float *x, const float *loss_scale,
                                            const float *grad_scale, float *loss, float *dx,
                                            BwppMeanSquareParams params);

/* BWPP_GOP_REDUCE_SUM / reduce_to_shape (graph_ir.c:1410-1455): axis 0 sums
 * over rows (out[cols]), any other axis along each row (out[rows]). */
BwppHipStatus bwpp_hip_dispatch_reduce_sum(BwppHip *h, const float *x, float *out,
                                           BwppReduceParams params);

/* add / sub / mul / div with broadcasting, and broadcast (op COPY). */
BwppHipStatus bwpp_hip_dispatch_elementwise(BwppHip *h, const float *a, const float *b, float *out,
                                            BwppElementwiseParams params);

/* ---- around the block: positions, residual joins ----
 * F32 or BF16 operands; arithmetic and sums in fp32, each output rounded
 * once.  With no rows (tokens) operands may be NULL, as empty tensors are, and
 * sums over rows are 0.  No reference counterparts. */

/* qo, ko = the rotated q, k.  positions: device int32 [batch][tokens] (row
 * stride pos_batch_stride) or NULL; any int32 is a position.  k may be NULL
 * with k_heads 0 (and q with q_heads 0).  qo may be q with the same strides
 * (in place; columns past rot_dim stay), and ko k; outputs must not meet
 * inputs or each other otherwise (ALIAS).  Angles are reduced in 64 bits. */
BwppHipStatus bwpp_hip_dispatch_rotary(BwppHip *h, const void *q, const void *k, const int32_t *positions, void *qo,
                                       void *ko, BwppRotaryParams params);

/* Its gradient: dq, dk (q's and k's strides) from dqo, dko (qo's and ko's):
 * the same turn backwards, the same magnitude. */
BwppHipStatus bwpp_hip_dispatch_rotary_grad(BwppHip *h, const void *dqo, const void *dko, const int32_t *positions,
                                            void *dq, void *dk, BwppRotaryParams params);

/* r and y of BwppResidualNormParams.  post_gamma, gate, pre_gamma NULL = 1
 * (gate NULL: no gate); y NULL: no norm after.  r may be x; outputs must not
 * meet inputs or each other otherwise (ALIAS).  y is taken from r before its
 * rounding. */
BwppHipStatus bwpp_hip_dispatch_residual_norm(BwppHip *h, const void *x, const void *o, const void *post_gamma,
                                              const void *gate, const void *pre_gamma, void *r, void *y,
                                              BwppResidualNormParams params);

/* Its gradient from the branch o, the stored r, and the upstream dr (of r, by
 * later blocks) and dy, either NULL = 0: dx (may be dr), dout (of o) and the
 * sums dpost_gamma [cols], dgate (gate's shape and row stride), dpre_gamma
 * [cols]; a NULL output is not computed.  Sums over rows are taken in fp32, in
 * an order that depends on the sizes only; their partial rows lie in the
 * handle's workspace. */
BwppHipStatus bwpp_hip_dispatch_residual_norm_grad(BwppHip *h, const void *o, const void *r, const void *post_gamma,
                                                   const void *gate, const void *pre_gamma, const void *dr,
                                                   const void *dy, void *dx, void *dout, void *dpost_gamma,
                                                   void *dgate, void *dpre_gamma, BwppResidualNormParams params);

/* loss[t] = lse[t] - z[t][targets[t]], lse[t] = log sum_v exp z[t][v] (natural,
 * fp32) for the logits of BwppLinearXentParams.  A target outside [0, vocab)
 * leaves its row out (loss 0, no gradient; its lse is still written).  sums
 * (may be NULL): [0] the sum of the losses, [1] how many rows count.  loss and
 * lse may be NULL, not all three.  bf16 needs dim >= 8 (and, W not transposed,
 * vocab >= 8).  fp32 products run on fp32 matrix instructions or, for more
 * tokens, on bf16 ones with each operand as three bf16 terms (24 bits).
 * Workspace: a pair of floats per row and 64 to 256 columns of the vocabulary;
 * fp32: the logits of a piece of it (256 MiB or 1024 columns), or terms of x and
 * of a piece of W (8 bytes an element; the piece in 256 MiB, up to 1 GiB for few
 * rows). */
BwppHipStatus bwpp_hip_dispatch_linear_xent(BwppHip *h, const void *x, const void *w, const int32_t *targets,
                                            float *loss, float *lse, float *sums, BwppLinearXentParams params);

/* Its gradients dx and dw (either may be NULL) for the upstream gradient dloss
 * of the row losses ([rows], one value with dloss_scalar, NULL = 1) and the
 * forward's lse.  The logits are made again, a piece of the vocabulary at a
 * time; bf16 rounds each dz to bf16 for the products that give dx and dw, whose
 * sums are fp32, and adds to them what that took from the targets' dz (not to
 * dx for a vocab below 8, nor to dw for a dim or a vocab of 2^23 and more).  A
 * dz that overflows to an infinity may come out as NaN.  dx rows of left-out tokens are 0, and their x
 * (which may hold anything) has no part in dw.  Outputs must not meet inputs or
 * each other (ALIAS).  Workspace: a copy of x, dz of a piece (256 MiB or 1024
 * columns, in some cases as many again), a float per row, and fp32 sums of dx
 * and of a small dw's piece, 1 to 32 planes each (the copy and a plane of dx
 * are rows x dim: they grow with the batch, whatever the piece); fp32 in terms:
 * those of x, W's and dz's piece, sums of dx and, up to 8 planes, of dw's
 * piece. */
BwppHipStatus bwpp_hip_dispatch_linear_xent_grad(BwppHip *h, const void *x, const void *w, const int32_t *targets,
                                                 const float *lse, const float *dloss, void *dx, void *dw,
                                                 BwppLinearXentParams params);

/* ---- a paged cache, and the next token ----
 * Operands and lengths of BwppCacheParams; no call reads lengths on the host.
 * With no tokens or no sequences operands may be NULL.  No reference
 * counterparts. */

/* Appends: k and v go to their slots, k and q with rotary positions, q to qo (may
 * be q with the same strides: in place; NULL with q_heads 0).  A token's position
 * is positions[row] (int32 [tokens]) or, NULL, its slot.  The rows of a pool must
 * not overlap, outputs must not meet inputs or each other otherwise (ALIAS).  Two
 * sequences with a page in common that write the same slot of it leave either's
 * rows. */
BwppHipStatus bwpp_hip_dispatch_cache_append(BwppHip *h, const void *q, const void *k, const void *v,
                                             const int32_t *positions, const int32_t *table, const int32_t *starts,
                                             const int32_t *held, void *qo, void *k_cache, void *v_cache,
                                             BwppCacheAppendParams params);

/* Attention of the new tokens, whose keys are in the cache already: token i of a
 * sequence sees the held tokens and those new tokens j whose bit j % 32 of word
 * j / 32 of its mask row (uint32 [tokens][mask_words]; bits past the row: not
 * seen) is set, or, without a mask, j <= i.  Query head h reads key head h /
 * (q_heads / heads).  o = softmax(scale q k) v; lse (may be NULL) [tokens][q_heads]
 * fp32 is the natural log-sum-exp.  A token that sees nothing gets 0 and -inf.
 * What lies in slots that a token does not see has no part in it, infinities and
 * NaN included.  Scores, sums and the probabilities that lse has are fp32.  With bf16
 * operands the probabilities enter the product with v as two bf16 terms (2^-16 of
 * each) or in fp32; for dim 128 and more than 32 rows rounded to one term (2^-8), as
 * attention's of that dim and as many queries are.  Rows are those of a sequence and
 * key head on average: `tokens` (rows of no sequence too) by `batch` (idle sequences
 * too), rounded up, times q_heads / heads; they also choose the kernel, one for all
 * sequences of a call.  Workspace: two partial results for each of one or two blocks a
 * compute unit, 16 to 256 rows of dim + 2 floats each (at most 65 MiB on 256 of them),
 * whatever the lengths. */
BwppHipStatus bwpp_hip_dispatch_cache_attention(BwppHip *h, const void *q, const void *k_cache, const void *v_cache,
                                                const int32_t *table, const int32_t *starts, const int32_t *held,
                                                const uint32_t *mask, void *o, float *lse,
                                                BwppCacheAttentionParams params);

/* After a tree of drafts is verified: slot held[s] + i takes the keys and values of
 * slot held[s] + kept[s][i] for i < counts[s] (int32 [batch], cut to max_kept), as
 * if all were read before any is written.  Of kept (int32 [batch][max_kept])
 * entries past the 16th must not be below their index (ascending ones are not);
 * entries below 0 or past the table move nothing.  Two sequences with a page in
 * common that write the same slot of it leave either's rows.  held itself is the
 * caller's to raise by counts. */
BwppHipStatus bwpp_hip_dispatch_cache_keep(BwppHip *h, void *k_cache, void *v_cache, const int32_t *table,
                                           const int32_t *held, const int32_t *kept, const int32_t *counts,
                                           BwppCacheKeepParams params);

/* y = x under the rules, row by row, in fp32.  Row r's history is history[starts[r]
 * .. starts[r + 1] - 1] (int32 tokens; those outside the vocabulary do not count),
 * its first prompt[r] (NULL: 0) given, the rest written.  In this order:
 *   z > 0 ? z / repetition[r] : z repetition[r]   where the token occurs
 *   z - (frequency[r] count + presence[r])        where it was written count times
 *   z + bias                                      fp32, row r of it or its one row
 *   -inf                                          where its mask bit (bit v % 32 of
 *                                                 word v / 32) is 0
 * NULL: without that rule.  y may be x (same dtype and stride), and must not meet
 * another operand otherwise (ALIAS). */
BwppHipStatus bwpp_hip_dispatch_logit_rules(BwppHip *h, const void *x, const int32_t *history, const int32_t *starts,
                                            const int32_t *prompt, const float *repetition, const float *presence,
                                            const float *frequency, const float *bias, const uint32_t *mask, void *y,
                                            BwppLogitRulesParams params);

/* ---- launch plans (compiled graphs) ----
 *
 * The executor for a lowered BW++ graph: `bwppc` hands its graph to the
 * Metal codegen today (main.c:186, codegen_metal.h:7); a HIP target emits
 * this text instead (format in csrc/runtime/bwpp_plan.cpp: dims, named
 * values, strided views, ordered operator launches over the dispatch calls
 * above).  Creation parses and builds the memory plan: liveness-based
 * buffer reuse as compiler/mem_plan.c:43-146, with byte sizes from the
 * bound dims and no operator ever given the buffer of one of its own
 * inputs.  h may be NULL to parse and plan only (report, arena size).
 * On failure *out still receives a plan whose last_error says why; destroy
 * it. */
typedef struct BwppHipPlan BwppHipPlan;
BwppHipStatus bwpp_hip_plan_create(BwppHip *h, const char *text, BwppHipPlan **out);
void bwpp_hip_plan_destroy(BwppHipPlan *plan);
const char *bwpp_hip_plan_last_error(const BwppHipPlan *plan);
/* Device bytes of all planned buffers (temps, outputs, consts). */
size_t bwpp_hip_plan_arena_bytes(const BwppHipPlan *plan);
/* One device arena (bwpp_hip_arena_init) holding every planned buffer;
 * const values are filled. */
BwppHipStatus bwpp_hip_plan_allocate(BwppHipPlan *plan);
/* Caller memory for an input or param value. */
BwppHipStatus bwpp_hip_plan_bind(BwppHipPlan *plan, const char *name, void *device_ptr);
/* Device address of any value (NULL if unknown or not yet placed). */
void *bwpp_hip_plan_value_ptr(const BwppHipPlan *plan, const char *name);
/* Runs every launch in order on the handle's stream. */
BwppHipStatus bwpp_hip_plan_run(BwppHipPlan *plan);
/* Records the plan's launches as a HIP graph (no reference counterpart: for
 * loops that replay one plan and should not pay the host cost of each
 * launch).  Runs the plan once eagerly first, so every workspace reaches its
 * final size, then captures one run on the handle's stream, which must not
 * be the default (null) stream (UNSUPPORTED).  The eager run is a run like any
 * other: cache_keep moves tokens on it, and what is written in place stays so.
 * Binding a different address afterwards drops the graph; capture again. */
BwppHipStatus bwpp_hip_plan_capture(BwppHipPlan *plan);
/* Launches the captured graph on the handle's current stream (INVALID_ARG
 * when there is none).  Results equal bwpp_hip_plan_run's.  Where the graph
 * uses the handle's scratch and its last use cannot be waited for (see
 * bwpp_hip_set_stream), runs the plan's launches instead. */
BwppHipStatus bwpp_hip_plan_replay(BwppHipPlan *plan);
/* Memory-plan report in mem_plan.c:176-193's layout plus byte sizes, arena
 * offsets and the total; returns the bytes needed including the NUL. */
size_t bwpp_hip_plan_report(const BwppHipPlan *plan, char *buf, size_t cap);

/* ---- synthetic inputs (host memory, no device needed) ----
 * Counter-based: element i of (seed, stream) is a pure function of
 * (seed, stream, i), so subsets and threads agree with a full fill.
 * SplitMix64 -> 24-bit uniform; normal by Box-Muller in double. */
void bwpp_synth_uniform_f32(float *dst, uint64_t n, uint64_t seed,
                            uint64_t stream, float lo, float hi);
void bwpp_synth_normal_f32(float *dst, uint64_t n, uint64_t seed,
                           uint64_t stream, float mean, float stddev);
/* The reference's test fixture x[i][j] = (i*cols + j + 1) * scale
 * (runtime/cpu/test_matmul.c:7-13). */
void bwpp_synth_ramp_f32(float *dst, uint32_t rows, uint32_t cols,
                         float scale);
/* fp32 -> bf16 round to nearest even (NaN kept quiet), and back (exact). */
void bwpp_f32_to_bf16(const float *src, uint16_t *dst, uint64_t n);
void bwpp_bf16_to_f32(const uint16_t *src, float *dst, uint64_t n);

#ifdef __cplusplus
}
#endif

#endif /* BWPP_HIP_H */

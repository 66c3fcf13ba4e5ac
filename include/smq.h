/* smq.h - C ABI of the MI355X (gfx950) quantized matrix-product path.
 *
 * A drop-in for the reference's kernel seam (src/kernels.h in
 * ktfth/smolmoe-c99): activation quantization to Q8, Q8 and Q5 weight rows
 * against Q8 activations (dot, 4-token, 4-row and gemm variants), the fused
 * matmul of up to four matrices sharing one input with bias and a finiteness
 * check (src/model.c:236-310), and row dequantization for embeddings.
 *
 * Conventions
 *  - Every array argument is a DEVICE pointer (hipMalloc'd or from smq_malloc)
 *    unless its comment says "host".
 *  - Work is enqueued on the library stream (smq_stream / smq_set_stream) and
 *    is ordered like any other work on that stream. Functions that return a
 *    computed value (smq_quantize_q8, smq_dot_q8, smq_dot_q5) synchronize.
 *  - Block layouts are the reference's on-disk layouts (docs/FORMAT.md:124-150):
 *    Q8 block = f32 LE scale + int8[32] (36 B); Q5 block = f16 LE scale + u32 LE
 *    high-bit plane + 16 nibble bytes (22 B); value = scale * (q - 16).
 *  - Results follow the reference's arithmetic contract (docs/FORMAT.md:152-171):
 *    exact int32 lane sums of 4 products, per lane acc = acc + (ws*xs)*lane in
 *    increasing block order (a single fmaf per lane in fast mode), then
 *    ((l0+l4)+(l2+l6)) + ((l1+l5)+(l3+l7)). Every smq_gemm_* output is bit
 *    identical to the reference's scalar kernel, except smq_gemm_*_mfma, whose
 *    per-block int32 sums are exact but whose f32 block order differs.
 *  - Errors: functions return or record an smq_status (the reference's
 *    sm_status values, src/util.h:28-37); smq_last_status / smq_last_error give
 *    the calling thread's latest failure (src/util.h:44-47).
 */
#ifndef SMQ_H
#define SMQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SMQ_QK 32u
#define SMQ_Q8_BLOCK_BYTES 36u /* kernels.h:46 */
#define SMQ_Q5_BLOCK_BYTES 22u /* kernels.h:47 */

/* src/util.h:28-37 */
typedef enum smq_status {
    SMQ_OK = 0,
    SMQ_ERR = 1,
    SMQ_ERR_IO = 2,
    SMQ_ERR_FORMAT = 3,
    SMQ_ERR_RANGE = 4,
    SMQ_ERR_NUMERIC = 5,
    SMQ_ERR_NOMEM = 6,
    SMQ_ERR_STATE = 7
} smq_status;

/* The calling thread's latest status and message (src/util.h:44-47). */
smq_status smq_last_status(void);
const char *smq_last_error(void);
void smq_clear_error(void);
/* Records a status and message for the calling thread, as sm_set does
 * (src/util.h:40-43), so host code layered on this library (the forward pass
 * in smq_model.h) reports through the same smq_last_error. Returns status. */
smq_status smq_set_error(smq_status status, const char *message);

/* ---- context ------------------------------------------------------------
 * One device per process (the reference's kernel table is process-global,
 * src/kernels.c:20-27). smq_init selects the device, checks it is gfx950 and
 * creates the library stream. */
smq_status smq_init(int device);
void smq_shutdown(void);
void *smq_stream(void);                      /* hipStream_t */
/* NULL restores the library stream. Decode attention at head size 64 has a workspace for the library's stream and two
 * of the caller's at a time; another one gets it after smq_synchronize, a copy or smq_numeric_check on its stream, and
 * computes the same without it. */
smq_status smq_set_stream(void *hip_stream);
smq_status smq_synchronize(void);
/* Device name of the selected GPU, e.g. "gfx950". */
const char *smq_device_arch(void);

/* ---- backend selection (src/kernels.h:72-87) -----------------------------
 * smq_kernels_select installs the GPU kernels behind the smq_* entry points
 * and returns the backend name: "gfx950" (exact mul+add contract) or
 * "gfx950-fast" (lane-wise FMA, kernels.h:9-11). force_exact ignores fast. */
const char *smq_kernels_select(int force_exact);
void smq_kernels_set_fast(int fast); /* kernels.h:77 */
int smq_kernels_fast(void);          /* kernels.h:78 */
/* kernels.h:72-73. The GPU kernels need no caller scratch: returns 0, and
 * every smq_gemm_* accepts scratch == NULL (a non-NULL scratch is ignored). */
size_t smq_gemm_scratch_bytes(uint32_t nb);
/* Host-side bounds checks of every operand range against its device
 * allocation before a launch (no reference counterpart). On by default, or
 * off when the environment sets SMQ_CHECKS=0. Ranges inside smq_malloc
 * allocations are checked against the library's own record; other device
 * memory through the runtime, except during a capture, where such ranges are
 * taken as given (no runtime call runs inside a capture). */
void smq_set_checks(int on);

/* ---- activation quantizer (src/kernels.h:183-187, kernels.c:912-935) ---- */
/* QuantizeQ8: n floats -> ceil(n/32) f32 scales d and 32*ceil(n/32) int8 q,
 * padding zero. Synchronous. Returns 0, or -1 if any input is inf or NaN (then
 * d and q are unspecified, as the reference's caller never reads them). */
int smq_quantize_q8(const float *x, uint32_t n, float *d, int8_t *q);
/* The caller's per-token loop (model.c:354-370): `rows` rows of n floats,
 * row r at x + r*n, into d + r*nb and q + r*nb*32. Asynchronous: a non-finite
 * input raises the sticky numeric flag read by smq_numeric_check. */
smq_status smq_quantize_q8_rows(const float *x, uint32_t rows, uint32_t n, float *d, int8_t *q);

/* ---- activation producers (src/model.c:347-415, src/vecmath.c:61-93) ----
 * The caller's per-token row work (row_work, model.c:354-362) for `rows` rows
 * of n floats (n <= 16384): optional RMSNorm with weight `norm` (NULL: none)
 * and eps (model.c:334-342, sequential f32 sum of squares); optional gated
 * activation with `gate` (act 0 = none, 1 = SwiGLU vecmath.c:78-81,
 * 2 = GeGLU vecmath.c:86-93, both with the deterministic binary64 exp of
 * vecmath.c:61-76); the f32 result stored to y when y != NULL (y may alias
 * src, as silu_quantize updates m->up in place); then quantize_q8 into
 * d + r*nb, q + r*nb*32. Bit-identical to the reference. A non-finite sum,
 * scale or value raises the sticky numeric flag. Asynchronous. */
smq_status smq_row_quantize(const float *src, const float *norm, float eps, const float *gate, int act, uint32_t rows,
                            uint32_t n, float *y, float *d, int8_t *q);
/* norm_quantize (model.c:393-400): RMSNorm then quantize. */
smq_status smq_norm_quantize(const float *src, const float *norm, float eps, uint32_t rows, uint32_t n, float *y,
                             float *d, int8_t *q);
/* silu_quantize (model.c:409-415): up *= act(gate) in place, then quantize;
 * gemma3 != 0 selects GeGLU. */
smq_status smq_silu_quantize(float *up, const float *gate, int gemma3, uint32_t rows, uint32_t n, float *d,
                             int8_t *q);

/* ---- dot products and gemm (src/kernels.h:49-70) -------------------------
 * Parameter lists are those of DotQ8, DotQ8x4, DotQ8R4 and GemmQ8. out is a
 * device array; smq_dot_q8/q5 return the value (synchronous). */
float smq_dot_q8(const unsigned char *w, const float *xd, const int8_t *xq, uint32_t nb);
float smq_dot_q5(const unsigned char *w, const float *xd, const int8_t *xq, uint32_t nb);
void smq_dot_q8_x4(const unsigned char *w, const float *xd, const int8_t *xq, uint32_t nb, uint32_t stride,
                   float *out);
void smq_dot_q5_x4(const unsigned char *w, const float *xd, const int8_t *xq, uint32_t nb, uint32_t stride,
                   float *out);
void smq_dot_q8_r4(const unsigned char *w, size_t row_bytes, const float *xd, const int8_t *xq, uint32_t nb,
                   float *out);
void smq_dot_q5_r4(const unsigned char *w, size_t row_bytes, const float *xd, const int8_t *xq, uint32_t nb,
                   float *out);
/* GemmQ8: out[t*stride + r] = dot(row r, activation t); activation t at
 * xd + t*nb, xq + t*nb*32. Decode (ntok == 1) runs the bandwidth GEMV;
 * ntok > 1 runs the exact LDS-tiled GEMM. Asynchronous. */
void smq_gemm_q8(const unsigned char *w, size_t row_bytes, const float *xd, const int8_t *xq, uint32_t nrows,
                 uint32_t ntok, uint32_t nb, float *out, size_t stride, unsigned char *scratch);
void smq_gemm_q5(const unsigned char *w, size_t row_bytes, const float *xd, const int8_t *xq, uint32_t nrows,
                 uint32_t ntok, uint32_t nb, float *out, size_t stride, unsigned char *scratch);
/* Prefill GEMM on int8 MFMA (no reference counterpart for its order: the
 * reference has one order). The per-block int32 sums are exact; each output is
 * acc = fma(wscale*xscale, float(blocksum), acc) over blocks in order, which
 * matches the exact contract within 1e-5 relative (|err| <= 1e-5 * max|out|
 * over a token's outputs). Same parameters as GemmQ8. Asynchronous. */
void smq_gemm_q8_mfma(const unsigned char *w, size_t row_bytes, const float *xd, const int8_t *xq, uint32_t nrows,
                      uint32_t ntok, uint32_t nb, float *out, size_t stride, unsigned char *scratch);
void smq_gemm_q5_mfma(const unsigned char *w, size_t row_bytes, const float *xd, const int8_t *xq, uint32_t nrows,
                      uint32_t ntok, uint32_t nb, float *out, size_t stride, unsigned char *scratch);
/* The MFMA path's per-block int32 sums, sums[(t*nrows + r)*nb + b] (device),
 * for the bit-exact integer check (test entry point, no reference counterpart). */
void smq_block_sums(int q5, const unsigned char *w, size_t row_bytes, const int8_t *xq, uint32_t nrows,
                    uint32_t ntok, uint32_t nb, int32_t *sums);
/* Which kernel smq_matmul uses when ntok > 1: 0 = the exact GEMM (default,
 * bit-identical to the reference), 1 = the int8-MFMA GEMM. */
void smq_set_prefill_mfma(int on);
/* Tuning (no reference counterpart): rows per workgroup of the
 * one-launch decode GEMV, 1, 2, 4, 8 or 16 (every output unchanged), or 0 =
 * chosen per width and row count (the default). Any other value is refused
 * with SMQ_ERR_RANGE. */
smq_status smq_set_gemv_rows(int rows);
/* Tuning (no reference counterpart): which kernel the exact prefill GEMM
 * (smq_gemm_q8 / smq_gemm_q5 / smq_matmul with ntok > 1) takes: 0 = chosen by
 * shape (the default), 1 = the one whose lane sums run on the matrix cores,
 * 2 = the one whose lane sums run as v_dot4, 3 (4) = the matrix-core one with
 * each tile's eight lane sums split over two (four) waves. Every output is the
 * same, bit for bit. Any other value is refused with SMQ_ERR_RANGE. */
smq_status smq_set_exact_gemm(int mode);

/* ---- fused matmul with bias and finiteness (src/model.c:236-310) -------- */
/* QMat (model.h:15-19): a weight matrix in device memory. dtype 1 = Q8, 2 = Q5
 * (docs/FORMAT.md:101). */
typedef struct smq_qmat {
    const unsigned char *data;
    uint32_t rows, cols, nb, dtype;
    size_t row_bytes;
} smq_qmat;
/* MatItem (model.c:236-240): y[token*w->rows + row] = dot + bias[row].
 * accumulate != 0 adds the result into y instead (y = y + result: the
 * residual add_rows of model.c:452-455 fused into the store, model.c:540,
 * 643); the finiteness check still looks at the result before the add. */
typedef struct smq_mat_item {
    const smq_qmat *w; /* host pointer to the descriptor */
    const float *bias; /* device, may be NULL */
    float *y;          /* device */
    int accumulate;
} smq_mat_item;
#define SMQ_MAX_ITEMS 4
/* Up to SMQ_MAX_ITEMS matrices with the same nb sharing one quantized input,
 * in one launch. A non-finite output raises the sticky numeric flag.
 * Asynchronous; SMQ_ERR_STATE if the items differ in width (model.c:298). */
smq_status smq_matmul(const smq_mat_item *items, uint32_t n, const float *xd, const int8_t *xq, uint32_t ntok);
/* No reference counterpart (the reference runs such matrices one matmul
 * after another, e.g. its experts in routed_experts, model.c:587-606):
 * independent decode GEMVs (one token each) in one launch. Item i computes
 * y_i[r] = dot(w_i row r, x_i) (+ bias_i[r]; added into y_i when accumulate),
 * with its own quantized activation x_i = (xd_i, xq_i). All items share nb
 * and the weight format; every output is bit-identical to smq_matmul's.
 * Persistent workgroups stream all items' weights back to back. At most
 * SMQ_MAX_GROUP items; asynchronous; the numeric flag as smq_matmul. */
#define SMQ_MAX_GROUP 48
typedef struct smq_group_item {
    const smq_qmat *w;  /* host pointer to the descriptor */
    const float *bias;  /* device, may be NULL */
    float *y;           /* device */
    int accumulate;
    const float *xd;    /* device: nb scales */
    const int8_t *xq;   /* device: nb*32 values */
} smq_group_item;
smq_status smq_gemv_grouped(const smq_group_item *items, uint32_t n);
/* A plan of independent one-token Q8 GEMVs streamed by one launch (no
 * reference counterpart: the reference runs them one after another), for
 * more items than SMQ_MAX_GROUP and for 28- and 152-block rows together (the
 * 896- and 4864-wide projections of Qwen2.5-0.5B: a whole FFN step's 72
 * GEMVs in one launch). Every item: packed Q8 rows (row_bytes = nb*36) of
 * nb = 28 or 152 blocks, 16-byte aligned, 4-byte aligned activations; every
 * output bit-identical to smq_matmul's. smq_gemv_plan_create validates the
 * items, splits them over workgroups in proportion to their bytes and copies
 * the split to device memory the plan owns (synchronously; not under
 * capture). smq_gemv_plan_launch is one asynchronous launch that may be
 * captured; the numeric flag as smq_matmul. The items' buffers must outlive
 * the plan; destroy a plan after every graph that launches it. */
#define SMQ_MAX_PLAN_ITEMS 4096
typedef struct smq_gemv_plan smq_gemv_plan;
smq_status smq_gemv_plan_create(const smq_group_item *items, uint32_t n, smq_gemv_plan **plan);
smq_status smq_gemv_plan_launch(const smq_gemv_plan *plan);
void smq_gemv_plan_destroy(smq_gemv_plan *plan);
/* Synchronizes, then returns SMQ_ERR_NUMERIC (and clears the flag) if any
 * quantize or matmul since the last check saw a non-finite value. */
/* ---- fused decode matmuls (one token) --------------------------------------
 * The activation of a decode matmul formed inside the matmul's own launch:
 * norm_quantize + matmul (model.c:503-509, 636-638) and silu_quantize +
 * matmul (model.c:639-643) without the activation round trip. Outputs are
 * bit-identical to the two-call forms, which these calls fall back to where
 * a shape does not fit the fused kernel (then the Q8 blocks go to the
 * scratch buffers). */
#define SMQ_ACT_Q8 0   /* xd, xq: the quantized activation */
#define SMQ_ACT_NORM 1 /* RMSNorm of x with norm and eps (model.c:334-342), then Q8 */
#define SMQ_ACT_F32 2  /* Q8 of the f32 row x (kernels.c:912-935) */
typedef struct smq_act {
    int kind;
    uint32_t cols;          /* elements: the matrices' cols */
    const float *x;         /* NORM, F32: cols floats */
    const float *norm;      /* NORM: cols floats */
    float eps;              /* NORM */
    const float *xd;        /* Q8: ceil(cols/32) scales */
    const int8_t *xq;       /* Q8: ceil(cols/32)*32 values */
    float *xd_scratch;      /* NORM, F32: room for the Q8 blocks if the call falls back */
    int8_t *xq_scratch;
} smq_act;
/* smq_matmul of one token with the activation `act`. */
smq_status smq_matmul_act(const smq_mat_item *items, uint32_t n, const smq_act *act);
/* The gate/up pair of a dense FFN (model.c:636-640): h[r] = up[r] *
 * act(gate[r]) with act 1 SwiGLU, 2 GeGLU (vecmath.c:78-93), gate and up the
 * matmuls of `act` (same rows and cols, no bias); a non-finite gate or up
 * raises the numeric flag. gate_scratch (gate->rows floats) holds the gate
 * row if the call falls back. */
smq_status smq_matmul_glu(const smq_qmat *gate, const smq_qmat *up, const smq_act *act, int glu, float *h,
                          float *gate_scratch);
/* smq_matmul_glu followed by silu_quantize's quantization (model.c:409-415:
 * quantize_q8 of h): hd (ceil(rows/32) scales) and hq (32 per block) receive
 * h's Q8 blocks, h (may be NULL where the shape allows) the f32 values. On
 * packed 896-wide Q8 rows the whole step is one launch; other shapes take the
 * two-call form, which needs h. The numeric flag as smq_matmul_glu, plus a
 * non-finite h. */
smq_status smq_matmul_glu_q8(const smq_qmat *gate, const smq_qmat *up, const smq_act *act, int glu, float *h,
                             float *hd, int8_t *hq, float *gate_scratch);
smq_status smq_numeric_check(void);

/* ---- decoder pieces around the matmuls ----------------------------------
 * Device-resident steps of the reference's forward pass (src/model.c:425-542,
 * 669-677) and its greedy choice (src/sampler.c:57-63). `pos_dev`, when not
 * NULL, is a device int32 read by the kernel in place of pos0, so a captured
 * decode step replays at successive positions. */
typedef struct smq_attn_shape {
    uint32_t heads, kv_heads, head_dim; /* query heads, KV heads (heads % kv_heads == 0) */
    uint32_t rotary_pairs;              /* rotary_dim / 2 (config.c:25-47) */
    uint32_t window;                    /* sliding window, 0 = full causal (model.c:466-470) */
    uint32_t context;                   /* positions the caches hold */
} smq_attn_shape;
/* model.c:511-526: for each of ntok tokens at position p = pos0 + t, rotate
 * q[t] (heads*head_dim) and k[t] (kv_heads*head_dim) in place by the table
 * rows cos_table[p], sin_table[p] (rotary_pairs floats each, model.c:425-450),
 * then store k[t] and v[t] into keys[p] and values[p] (kv_heads*head_dim f32
 * each). A position at or past context raises the numeric flag instead. */
smq_status smq_rope_kv(float *q, float *k, const float *v, uint32_t ntok, const smq_attn_shape *shape,
                       const float *cos_table, const float *sin_table, float *keys, float *values, uint32_t pos0,
                       const int32_t *pos_dev);
/* model.c:459-491 with attend_f32 (kernels.c:1154-1176): causal attention of
 * each query head of ntok tokens over keys/values[start .. p], p = pos0 + t,
 * in the reference's order (8-lane dot, exp_det softmax, sums in position
 * order), writing att[t] (heads*head_dim). Bit identical to the reference. */
smq_status smq_attention(const float *q, const float *keys, const float *values, float *att, uint32_t ntok,
                         const smq_attn_shape *shape, uint32_t pos0, const int32_t *pos_dev);
/* smq_attention followed by quantize_attention (model.c:402-406): att rows
 * also quantized to Q8 into xd (ntok*nb f32) and xq (ntok*nb*32), nb =
 * ceil(heads*head_dim / 32); one launch when head_dim % 32 == 0. */
smq_status smq_attention_q8(const float *q, const float *keys, const float *values, float *att, uint32_t ntok,
                            const smq_attn_shape *shape, uint32_t pos0, const int32_t *pos_dev, float *xd,
                            int8_t *xq);
/* One decoding token (model.c:511-542 for ntok = 1): smq_rope_kv, then
 * smq_attention_q8, as one launch where the shape allows (head_dim 64,
 * 16-byte aligned q, k, v and caches; otherwise the two calls). q and k are the unrotated QKV outputs; afterwards their contents
 * are unspecified (rotated or not). keys/values[p] receive the rotated k and
 * v of this position, att the attention row, xd/xq its Q8 blocks. */
smq_status smq_attention_rope_q8(float *q, float *k, const float *v, const smq_attn_shape *shape,
                                 const float *cos_table, const float *sin_table, float *keys, float *values,
                                 float *att, uint32_t pos0, const int32_t *pos_dev, float *xd, int8_t *xq);
/* The q, k, v matmuls of one decoding token (items[0..2], rows q_dim, kv_dim,
 * kv_dim, no accumulate) with the activation `act`, followed by RoPE and the
 * cache store (model.c:496-526): the same results as smq_matmul_act then
 * smq_rope_kv(items[0].y, items[1].y, items[2].y, 1, ...), i.e. q and k rotated
 * by the position's table rows (model.c:442-450) in their outputs, and the
 * rotated k and the v row written into keys/values at the position (pos_dev if
 * not NULL, else pos0). Q8 rows of 28 blocks with an RMSNorm activation do it in
 * one launch. No reference counterpart of its own: it fuses the two calls above,
 * each of which has one. */
smq_status smq_matmul_act_rope(const smq_mat_item *items, const smq_act *act, const smq_attn_shape *shape,
                               const float *cos_table, const float *sin_table, float *keys, float *values,
                               uint32_t pos0, const int32_t *pos_dev);
/* sampler.c:57-63: *token = first non-banned id, replaced by any later
 * non-banned id with a strictly greater logit (NaN never wins unless it is
 * the first candidate). banned may be NULL. UINT32_MAX if every id is banned. */
smq_status smq_argmax(const float *logits, uint32_t vocab, const unsigned char *banned, uint32_t *token);
/* No counterpart in the reference. For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): smq_argmax with its partial results in a static device
 * array of the library (12 KiB per GPU, bound at smq_init) instead of the
 * library's allocated workspace; it calls no allocation routine. Same result
 * as smq_argmax. vocab is limited to 1,048,576 ids (SMQ_ERR_RANGE beyond).
 * Every call on one GPU shares that array: calls that overlap on one GPU
 * (different streams, or concurrent host threads) race. Asynchronous. */
smq_status smq_argmax_noalloc(const float *logits, uint32_t vocab, const unsigned char *banned, uint32_t *token);
/* model.c:669-677: x[t] = dequantized row tokens[t] of the embedding matrix
 * (embed->cols floats). Ids must be < embed->rows (checked by the caller, as
 * model.c:671-672 does; an id out of range raises the numeric flag). */
smq_status smq_embed(const smq_qmat *embed, const uint32_t *tokens, uint32_t ntok, float *x);
/* Decode-loop bookkeeping on the device: history[*count] = *token when
 * *count < capacity, then ++*count and ++*pos (lets a captured step advance). */
smq_status smq_decode_advance(int32_t *pos, uint32_t *count, const uint32_t *token, uint32_t *history,
                              uint32_t capacity);
/* smq_argmax then smq_decode_advance in one call (the greedy step of the
 * reference's generation loop, main.c:580-600, on device state). Calls on one
 * stream share the library's argmax workspace; concurrent calls on different
 * streams race. */
smq_status smq_argmax_advance(const float *logits, uint32_t vocab, const unsigned char *banned, uint32_t *token,
                              int32_t *pos, uint32_t *count, uint32_t *history, uint32_t capacity);
/* smq_argmax_advance, then the chosen token's embedding row into x
 * (embed->cols floats): the next decode step's input (model.c:669-677), so a
 * captured step needs no embedding launch of its own. No reference
 * counterpart: it fuses the greedy pick (sampler.c:57-63) with the next
 * step's smq_embed. An id past the vocabulary (every id banned) raises the
 * numeric flag instead of writing x, as smq_embed does. */
smq_status smq_argmax_advance_embed(const float *logits, uint32_t vocab, const unsigned char *banned, uint32_t *token,
                                    int32_t *pos, uint32_t *count, uint32_t *history, uint32_t capacity,
                                    const smq_qmat *embed, float *x);

/* ---- paged KV cache: several sequences at once -----------------------------
 * No reference counterpart (the reference holds one sequence in one f32 or f16
 * cache, src/model.h:59-61): the caches of many sequences in pages of one
 * pool, and batches of sequences that bring different numbers of new tokens
 * (one while decoding, a chunk of a prompt). One pool pair holds one layer.
 *
 * A page holds page_size positions of every KV head: keys as
 * [kv_head][position][head_dim], values as [kv_head][head_dim][position].
 * SMQ_KV_Q8 holds int8 codes and an f32 scale per position and 32-wide block
 * of a head, [kv_head][ceil(head_dim / 32)][position] per page: the activation
 * quantizer's rule (smq_quantize_q8) over each head's dims, the last block
 * shorter where head_dim is no multiple of 32. */
#define SMQ_KV_F32 0u
#define SMQ_KV_F16 1u
#define SMQ_KV_Q8 2u
typedef struct smq_paged_kv {
    void *keys, *values;              /* device, 16-byte aligned: `pages` pages each */
    float *key_scales, *value_scales; /* device, 16-byte aligned, SMQ_KV_Q8 only */
    uint32_t type;                    /* SMQ_KV_* */
    uint32_t page_size;               /* positions of a page: 16, 32, 64, 128 or 256 */
    uint32_t pages;
} smq_paged_kv;
/* A batch of seqs sequences. The new tokens' rows lie one after another: those
 * of sequence s are rows begin[s] .. begin[s + 1] - 1, n of them (0 allowed),
 * and row begin[s] + i stands at position length[s] - n + i. Positions x of
 * sequence s lie in page table[s * table_stride + x / page_size]. The arrays
 * are read on the device, so a captured launch replays with new contents.
 * Rows before begin[0] and from begin[seqs] on are padding: never read, never
 * written.
 *
 * What the host cannot check raises the sticky numeric flag on the device and
 * touches nothing out of range: a page id outside [0, pages) (only of a page
 * that the call needs), a row whose position is negative, at or past
 * shape->context or past the table (not stored, not read, its attention is
 * 0), a begin that does not ascend within 0 .. tokens (which rows are computed
 * is then unspecified). Rows in such pages are not stored and not read,
 * positions in them not seen.
 *
 * Refused: more than 1,048,576 sequences or pages of a sequence, and tokens
 * times shape->heads above 4,194,304. */
typedef struct smq_paged_batch {
    const int32_t *begin;  /* device, seqs + 1 */
    const int32_t *length; /* device, seqs: positions including the new tokens */
    const int32_t *table;  /* device, seqs * table_stride page ids */
    uint32_t seqs, tokens, table_stride;
} smq_paged_batch;
/* smq_rope_kv for a paged cache: every new token's k (kv_heads * head_dim
 * floats a row) rotated by its position's table row (rotary_pairs floats each,
 * shape->context rows) and v into the cache as kv->type holds them; k itself
 * is left as it is. q's rows, rotated, go to q_out (q_out == q rotates in
 * place; both NULL: none). Rotation as smq_rope_kv's, bit for bit; f16
 * rounds to nearest even. A value that the type cannot hold as a finite number
 * raises the numeric flag (f16: infinite; Q8: its block gets a NaN scale).
 * Sequences must not share a page that the call writes to. shape: head_dim a
 * multiple of 16, at most 256, context at most 1,048,576. Asynchronous. */
smq_status smq_paged_rope_kv(const float *q, float *q_out, const float *k, const float *v,
                             const smq_paged_batch *batch, const smq_attn_shape *shape, const float *cos_table,
                             const float *sin_table, const smq_paged_kv *kv);
/* The batch's rows out of the cache as f32: keys and values row r =
 * kv_heads * head_dim floats, what the cache holds at the row's position (f16
 * exactly, Q8 code * scale). With begin the running sum of length, whole
 * sequences, for instance into contiguous caches. Asynchronous. */
smq_status smq_paged_read(const smq_paged_batch *batch, const smq_attn_shape *shape, const smq_paged_kv *kv,
                          float *keys, float *values);
/* Attention of the new tokens (their keys and values are in the cache): head h
 * of the row at position p over the positions j <= p of its sequence, with
 * shape->window w > 0 only those with j > p - w or j < sinks:
 *   att[h] = sum_j softmax_j(q[h] . k[j] / sqrt(head_dim)) v[j]
 * (KV head h / (heads / kv_heads)); f32 sums and statistics, each product of
 * f32 accuracy, where the cache is not f32 down to 2^-31 of the row's largest
 * weight (Q8: of that times the largest scale that the row sees of the value's
 * 32 dims, 2^-112 at least), no order of the sums promised beyond: the same call
 * gives the same bits. Values of up to 3.3e38 give finite results. A row that
 * sees nothing is 0. Keys and values at positions that a row does not see, and
 * slots past a sequence's length, never matter, NaN and infinities included; a
 * visible one that is not finite leaves the row's result unspecified. Pages that
 * no row sees may have any id. att must not overlap q.
 * workspace (device, 16-byte aligned, may be NULL): where the call splits long
 * sequences over workgroups, their partial results;
 * smq_paged_attention_workspace gives the bytes that allow the widest split
 * with any number of sinks, fewer bytes split less. Whether to split at all the
 * host decides by shape->context, the table's width, the window and the sinks: a
 * context near the longest length saves short batches a launch. Calls that may
 * overlap in time, replays of different graphs among them, must not share one.
 * Asynchronous, capturable. */
size_t smq_paged_attention_workspace(const smq_paged_batch *batch, const smq_attn_shape *shape);
smq_status smq_paged_attention(const float *q, float *att, const smq_paged_batch *batch, const smq_attn_shape *shape,
                               uint32_t sinks, const smq_paged_kv *kv, void *workspace, size_t workspace_bytes);

/* ---- drafted tokens and beams over the paged cache --------------------------
 * No reference counterpart (the reference decodes one sequence, one token at a
 * time): what goes on top of the paged cache where a step brings a tree of
 * drafted tokens for each sequence, or where sequences are the beams of a
 * search and share pages. */
/* The rows of smq_paged_norm_rope_kv. A stride is the floats from one token's
 * row to the next one's, 0 for rows one after another: q, k and v may be parts
 * of one wider row. */
typedef struct smq_paged_rows {
    const float *q;            /* heads * head_dim floats a row; NULL with q_out: none */
    float *q_out;              /* q itself with the same stride: in place */
    const float *k, *v;        /* kv_heads * head_dim floats a row */
    size_t q_stride, q_out_stride, k_stride, v_stride;
    const float *q_norm, *k_norm; /* head_dim floats each, device; NULL: no norm */
    float eps;                 /* finite, not negative */
    const int32_t *depth;      /* device, one per token: its rotary position is the number of positions before its
                                * sequence's new tokens + depth (drafts that continue the same token share a position);
                                * NULL: the position in the cache */
} smq_paged_rows;
/* smq_paged_rope_kv with an RMSNorm of each head of q and k before the
 * rotation and with rotary positions of the tokens' own:
 *   y = (x * (1 / sqrt(mean(x^2) + eps))) * norm
 * mean, root and quotient in 64 bits, the quotient and both products rounded
 * to f32 each (no order of the mean's sum shows in the result), then the
 * rotation and the cache's rounding as smq_paged_rope_kv has them. Keys and
 * values go to the tokens' own places whatever their depth. A row whose rotary
 * position is outside [0, context) raises the numeric flag: its k is not
 * stored and its q not written. q_out must not overlap what the call reads, but
 * for q in place. Asynchronous, capturable. */
smq_status smq_paged_norm_rope_kv(const smq_paged_rows *rows, const smq_paged_batch *batch, const smq_attn_shape *shape,
                                  const float *cos_table, const float *sin_table, const smq_paged_kv *kv);
/* Trees of drafted tokens: parent[r], for row r of the batch, is the index
 * among its sequence's new tokens of the token that r continues, below its own
 * index; negative where that is the last token of the context. depth[r]: 0
 * there, else its parent's + 1. mask, mask_stride words a row: bit t % 32 of
 * word t / 32 is set where t is the token itself or an ancestor; the other
 * bits of the row's words are cleared. A parent at or past its own index
 * raises the numeric flag and counts as negative. A sequence of more than
 * 32 * mask_stride new tokens raises the flag; its rows are left as they are,
 * as those of padding. mask_stride: 1 .. 128. One call serves the attention of
 * all layers. depth and mask must not overlap each other, parent or begin.
 * Asynchronous, capturable. */
smq_status smq_draft_masks(const int32_t *parent, const smq_paged_batch *batch, int32_t *depth, uint32_t *mask,
                           uint32_t mask_stride);
/* smq_paged_attention where a mask says which of its sequence's new tokens a
 * row sees: of the positions before them (the context) all, with shape->window
 * w > 0 those with j > p - w or j < sinks, p = the context's positions +
 * depth[r] (not read where there is no window); of the new tokens those whose
 * bit is set, whatever the window, later ones too (smq_draft_masks knows no
 * window: where drafts reach as deep as one, the caller clears the bits of the
 * ancestors w or more levels above that are no sinks, and a chain's attention
 * is smq_paged_attention's). mask as smq_draft_masks writes it, or any other:
 * bits behind the last new token, and of those without a place, do not matter.
 * A row that sees nothing is 0. Numbers, errors, workspace and what does not matter
 * as smq_paged_attention's; a depth below 0 or where p is not below the
 * context's size raises the numeric flag, its row is 0, and so are those of a
 * sequence of more than 32 * mask_stride new tokens. All pages of the new
 * tokens must be pages. mask_stride: 1 .. 128. att must not overlap q, depth
 * or mask. The workspace has a query of its own. Asynchronous, capturable. */
size_t smq_paged_tree_attention_workspace(const smq_paged_batch *batch, const smq_attn_shape *shape);
smq_status smq_paged_tree_attention(const float *q, float *att, const smq_paged_batch *batch, const smq_attn_shape *shape,
                                    uint32_t sinks, const int32_t *depth, const uint32_t *mask, uint32_t mask_stride,
                                    const smq_paged_kv *kv, void *workspace, size_t workspace_bytes);
/* The accepted path of each sequence's draft to the front of its new tokens,
 * in every pool (the layers' caches: same type, page_size and pages): for k
 * below count[s] the keys and values of new token accepted[s * accepted_stride
 * + k] go to the place of new token k, as the cache holds them. length_out[s]
 * = the positions before the new tokens + count[s]; it must not overlap the
 * batch's arrays, accepted or count. A list that does not ascend strictly
 * within the sequence's new tokens, or is longer than accepted_stride, raises
 * the numeric flag: the sequence stays as it is, its length too. Positions
 * without a place or page raise the flag and are not moved. Sequences must not
 * share a page that the call writes to. At most SMQ_MAX_POOLS pools; one that
 * is named again counts once, others that share memory are refused.
 * Asynchronous, capturable. */
#define SMQ_MAX_POOLS 1024u
smq_status smq_paged_compact(const smq_paged_batch *batch, const smq_attn_shape *shape, const int32_t *accepted,
                             uint32_t accepted_stride, const int32_t *count, const smq_paged_kv *pools, uint32_t n_pools,
                             int32_t *length_out);
/* The next page tables of a set of sequences: rows of the new table that go on
 * from rows of the old one. New row d keeps the first keep[d] positions of old
 * row parent[d] (-1: none, and nothing is kept) and gets pages for room[d]
 * positions in all (at least keep[d]):
 *  - pages that keep[d] fills are shared with every row that names them;
 *  - a page that it fills in part stays where nothing else holds it then (of
 *    several rows that take it in part the first one keeps it), else its
 *    positions are to be copied to a page of the row's own: copies[d];
 *  - further pages are free ones, the lowest ids in the order of rows and
 *    entries.
 * So one call forks sequences (a parent named twice), ends them (a parent not
 * named), begins them (-1), gives back what drafts have taken (keep below the
 * length) and makes room for the next tokens (room above it). Old arrays are
 * left as they are; no new one may overlap another array.
 *
 * refs counts, for each page, the entries of the old table (of the first
 * held[s] ones of each row) that name it and other holders (a store of
 * prompts), which stay counted; 0: free. refs_out: the same for the new table.
 * held_out[d] = ceil(room[d] / page_size); entries behind it are -1. copies:
 * three words a row, the page copied from and to and its positions; -1, -1, 0
 * where nothing is to be copied. free_out: the pages free afterwards; negative
 * where so many were missing (-2^31: so many or more): then the numeric flag is
 * raised, entries without a page are -1, and the old arrays still hold.
 *
 * Raise the flag as well: held, keep or room outside the table's row (cut), a
 * keep above the parent's pages (cut) or above room (room is raised), a parent
 * outside the old rows (-1), an entry that is no page (it stays none), refs
 * seen to be below the old table's entries (such a page may be given twice).
 * workspace: device, 16-byte aligned; calls that may overlap in time must not
 * share one. At most 65535 rows and 2^24 pages. Asynchronous, capturable. */
typedef struct smq_page_fork {
    const int32_t *table; /* old_seqs * table_stride page ids */
    const int32_t *held;  /* old_seqs: entries that hold pages */
    const int32_t *refs;  /* pages */
    uint32_t old_seqs, seqs, table_stride;
    uint32_t page_size, pages; /* as smq_paged_kv's */
    const int32_t *parent, *keep, *room; /* seqs */
    int32_t *table_out;   /* seqs * table_stride */
    int32_t *held_out;    /* seqs */
    int32_t *refs_out;    /* pages */
    int32_t *copies;      /* seqs * 3 */
    int32_t *free_out;    /* one word */
} smq_page_fork;
size_t smq_paged_fork_workspace(const smq_page_fork *fork);
smq_status smq_paged_fork(const smq_page_fork *fork, void *workspace, size_t workspace_bytes);
/* The copies of smq_paged_fork in every pool: of row i the first copies[3 i +
 * 2] positions of page copies[3 i] into page copies[3 i + 1], nothing else of
 * that page. No page may be written twice or be read and written. Ids that are
 * no page, or more positions than page_size, raise the numeric flag, and the
 * row is skipped; so is one of no positions, without the flag. shape: kv_heads
 * and head_dim. Pools as smq_paged_compact's. Asynchronous, capturable. */
smq_status smq_paged_copy(const int32_t *copies, uint32_t rows, const smq_attn_shape *shape, const smq_paged_kv *pools,
                          uint32_t n_pools);
/* A step of a beam search: `groups` of `beams` rows of logits each (row r at
 * logits + r * stride), and of each group the `select` best continuations,
 * best first. A continuation of row r by id v is worth
 *   score[r] + (l[v] - log sum_u exp(l[u]))
 * in 64 bits, sum and logarithm included (each exponential within 1e-12 of its
 * size); the results are rounded to f32. Equal ones: the lower row first; of
 * one row, the larger logit, then the lower id. A row that is done has one continuation, by `pad`,
 * worth score[r]. Continuations worth -inf (masked ids) are none. Where a
 * group has fewer than `select`, the rest gets parent -1, token UINT32_MAX,
 * score -inf and counts as done. A row that is not done with a NaN or +inf
 * among its logits, or any with a score that is NaN or +inf, raises the
 * numeric flag and has no continuation.
 *
 * parent[i] is the row in 0 .. groups * beams - 1, as smq_paged_fork takes it.
 * done_out[i]: the parent was done or the token is eos. History rows
 * (history_stride ids each, as many as `length` says): row i of history_out
 * has the parent's ids and, unless the parent was done, the token behind them
 * (a row that is full raises the numeric flag and stays as it is); the rest of
 * the row is UINT32_MAX, which smq_logits_adjust skips, so that history_begin
 * may be multiples of history_stride. Lengths outside [0, history_stride]
 * raise the flag and are cut. No new array may overlap another one.
 *
 * select and beams: 1 .. 64, vocab: at most 1,048,576, at most 65535 rows of
 * logits or of results. workspace: device, 16-byte aligned, the query's bytes,
 * which suffice for fewer rows, ids or results too; calls that may overlap in
 * time must not share one. Asynchronous, capturable. */
typedef struct smq_beam_step {
    const float *logits;
    size_t stride;
    uint32_t groups, beams, vocab, select;
    const float *score;         /* device, a row's own so far */
    const uint8_t *done;        /* device, a row's own; NULL: none is */
    uint32_t pad, eos;          /* eos UINT32_MAX: none */
    int32_t *parent;            /* groups * select each */
    uint32_t *token;
    float *score_out;
    uint8_t *done_out;          /* NULL: not wanted */
    const uint32_t *history;    /* groups * beams rows; NULL: no histories */
    uint32_t *history_out;      /* groups * select rows */
    uint32_t history_stride;
    const int32_t *length;      /* ids in each row */
    int32_t *length_out;
} smq_beam_step;
size_t smq_beam_select_workspace(const smq_beam_step *step);
smq_status smq_beam_select(const smq_beam_step *step, void *workspace, size_t workspace_bytes);

/* ---- logits of several rows before the choice of a token -------------------
 * No reference counterpart (sampler.c:57-63 only skips banned ids). For each
 * row, with c the times id v stands in the row's history:
 *   l = logits[v]
 *   c > 0: l = (l > 0 ? l / repetition : l * repetition) - (c * frequency + presence)
 *   l += the sum of the row's biases for v
 *   l = -inf where the row's mask does not allow v
 * and the greedy token: smq_argmax's choice (the lowest id on ties; a NaN only
 * where it is the first candidate) among the allowed ids, UINT32_MAX if there
 * is none. Ids at or past vocab in history and bias_ids are skipped. Lists end
 * at history_count and bias_count whatever the begin arrays say. */
typedef struct smq_logit_rules {
    const uint32_t *history;      /* device; NULL: no penalties */
    const int32_t *history_begin; /* device, rows + 1: row r's ids are history[history_begin[r]] .. */
    uint32_t history_count;
    const float *penalty;         /* device, rows x 3: repetition, presence, frequency (1, 0, 0: none) */
    const uint32_t *bias_ids;     /* device; NULL: no biases */
    const float *bias;            /* device: one for each of bias_ids */
    const int32_t *bias_begin;    /* device, rows + 1 */
    uint32_t bias_count;
    const uint32_t *allowed;      /* device, allowed_rows x ceil(vocab / 32) words, bit v % 32 of word v / 32; NULL: none */
    uint32_t allowed_rows;
    const int32_t *mask_row;      /* device, rows: the row of `allowed`, negative: no mask; NULL: row r of allowed.
                                   * An index at or past allowed_rows raises the numeric flag and allows nothing. */
} smq_logit_rules;
/* Row r of logits at logits + r * stride, of out at out + r * out_stride (out
 * may be logits with the same stride, must not overlap it otherwise; NULL: only
 * the tokens); token (rows, may be NULL when out is not). rules NULL: only the
 * choice. workspace (device, 16-byte aligned, smq_logits_workspace bytes, which
 * suffice for fewer rows or ids too) is needed with token; calls that may
 * overlap in time must not share one. Asynchronous, capturable. */
size_t smq_logits_workspace(uint32_t rows, uint32_t vocab);
smq_status smq_logits_adjust(const float *logits, size_t stride, uint32_t rows, uint32_t vocab,
                             const smq_logit_rules *rules, float *out, size_t out_stride, uint32_t *token,
                             void *workspace, size_t workspace_bytes);

/* ---- Q5 weight conversion (src/kernels.h:205, kernels.c:1064-1117) -------
 * quantize_q5_row: cols floats x -> ceil(cols/32) Q5 blocks (22 B each) at
 * out, byte for byte the reference's: signed extreme, the first minimum of 21
 * f16-rounded candidate scales by binary64 squared error, codes packed as in
 * docs/FORMAT.md:124-134. Device pointers, asynchronous. */
void smq_quantize_q5_row(const float *x, uint32_t cols, unsigned char *out);
/* The converter's loop over a tensor (src/quantize_main.c:107-121): `rows`
 * rows of cols floats (row r at x + r*cols) into rows of ceil(cols/32)*22
 * bytes (row r at out + r*ceil(cols/32)*22), one launch. */
smq_status smq_quantize_q5_rows(const float *x, uint32_t rows, uint32_t cols, unsigned char *out);

/* ---- dequantization (src/kernels.h:193-196, kernels.c:1044-1062) -------- */
void smq_dequantize_q8_row(const unsigned char *w, uint32_t cols, float *out);
void smq_dequantize_q5_row(const unsigned char *w, uint32_t cols, float *out);

/* ---- graph capture (no reference counterpart: amortizes launches) -------
 * Work enqueued on the library stream between smq_capture_begin and
 * smq_capture_end is recorded, not run, and replayed by smq_graph_launch
 * (a HIP graph). Only asynchronous entry points may be captured: smq_gemm_*,
 * smq_dot_*_x4/_r4, smq_matmul, smq_quantize_q8_rows, smq_dequantize_*, the
 * paged cache's, smq_logits_adjust and those of drafts and beams (batches,
 * rules, trees, parents and scores are read on the device at each replay; what
 * the host passed, tokens and context among it, stays). */
smq_status smq_capture_begin(void);
void *smq_capture_end(void);
smq_status smq_graph_launch(void *graph);
void smq_graph_destroy(void *graph);

/* ---- device memory and timing helpers (plumbing for C hosts and tests) -- */
void *smq_malloc(size_t bytes);
void smq_free(void *p);
smq_status smq_memcpy_htod(void *dst, const void *host_src, size_t bytes);
smq_status smq_memcpy_dtoh(void *host_dst, const void *src, size_t bytes);
smq_status smq_memcpy_dtod(void *dst, const void *src, size_t bytes);
smq_status smq_memset(void *dst, int value, size_t bytes);
/* Records a start event on the library stream. */
smq_status smq_timer_start(void);
/* Records a stop event, waits for it, returns milliseconds since start (<0 on error). */
double smq_timer_stop(void);

/* ---- cross-workgroup hand-off anchor (no reference counterpart: measurement)
 * One launch of `workgroups` workgroups (1..the device's CU count; each holds
 * 96 KB of LDS, so one per CU and all resident) passing `episodes` (<= 100000)
 * grid barriers, timed on the library stream into *ms (host). kind 0: one
 * counter, every workgroup adds 1 and waits for the generation's total; kind
 * 1: eight counters by workgroup index % 8 (the XCD the workgroup is dealt
 * to), the last arriver of each adds 1 to one release counter; kind 2: no
 * atomics, every workgroup stores the generation into a word of its own,
 * workgroup 0 waits for all of them and publishes it. Agent-scope release and
 * acquire. Every wait is bounded (2^20 polls), a workgroup that gives up ends
 * every other wait, and the call then returns SMQ_ERR_STATE. Synchronizes;
 * not for use under capture; allocates a 2.5 KB counter buffer once. */
smq_status smq_grid_barrier_probe(uint32_t workgroups, uint32_t episodes, uint32_t kind, double *ms);

/* ---- HBM bandwidth anchors (no reference counterpart: measurement) ------
 * Plain kernels that read (smq_stream_read) or copy (smq_stream_copy) `bytes`
 * (a multiple of 16, 16-byte aligned) with coalesced 16-byte loads, so a
 * GEMV's GB/s can be read against what the device's HBM delivers. A grid of
 * `workgroups` x `threads` (64..1024, a multiple of 64) threads; nontemporal
 * selects non-temporal loads and stores. The read writes nothing (`sink`, a
 * device word, is written only for one improbable data pattern).
 * Asynchronous, capturable. */
smq_status smq_stream_read(const void *p, size_t bytes, uint32_t workgroups, uint32_t threads, int nontemporal,
                           uint32_t *sink);
smq_status smq_stream_copy(void *dst, const void *src, size_t bytes, uint32_t workgroups, uint32_t threads,
                           int nontemporal);

#ifdef __cplusplus
}
#endif

#endif

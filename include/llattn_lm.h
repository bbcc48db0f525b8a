/* The ends and the feed-forward of the language model around the block: token
 * and position rows with their gradients, the gated feed-forward, the norm of
 * all gradients and their clipping.  Same conventions as llattn.h (status
 * codes, llattn_last_error, explicit stream, caller-supplied memory, nothing
 * allocated, no state kept between calls).  In the reference: nn.Embedding
 * twice and their sum (within models.py:505-580), clip_grad_norm_
 * (train.py:1021); its feed-forward (models.py:50-58) has no gate. */
#ifndef LLATTN_LM_H
#define LLATTN_LM_H

#include "llattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- token rows, scaled, plus position rows ---------------------------------
 *   out[n] = scale W[id_n] + Pos[pos_n]      in fp32, rounded once
 * for rows n < rows: W [V][D], Pos [P][D] (P = 0: none), out [rows][D], all of
 * `dtype`, row strides ldw and ldp in elements, any alignment of whole
 * elements.  ids and pos hold integers of index_bytes (4 or 8); pos NULL: pos_n
 * = n % T.  A row whose id lies outside [0, V), or whose position lies outside
 * [0, P), is NaN.
 *
 * Backward, from dout [rows][D] contiguous:
 *   dW[v] = scale sum of dout[n] over id_n = v (v != padding), dPos[p] = sum of
 *   dout[n] over pos_n = p,
 * whole tables [V][D] and [P][D], contiguous (rows that no token names are
 * zero), either NULL.  Rows of no valid id (position) leave dW (dPos) alone.
 * The rows of one token are summed in fp32 in their order, in a tree that the
 * number of them alone decides: no atomics, and the same bits whatever the
 * other tokens are.  It reads the order of the rows that llattn_embed_order has
 * written for the same configuration and indices, at any time before: by token
 * (`tokens`, where dW is wanted) and by position (`positions`, where pos is
 * given and dPos wanted). */
typedef struct llattn_embed_cfg {
  int64_t rows;         /* below 2^31 */
  int32_t T, V, P, D;   /* V and P at most 2^22 */
  int32_t dtype;        /* LLATTN_F32 or LLATTN_BF16 */
  int32_t index_bytes;
  int64_t padding;      /* a token without gradient, or -1 */
  float scale;          /* finite */
} llattn_embed_cfg;

int32_t llattn_embed_fwd(const llattn_embed_cfg* cfg, const void* ids, const void* pos, const void* W, int64_t ldw,
                         const void* Pos, int64_t ldp, void* out, void* stream);
/* Bytes of a buffer (1: none is needed, NULL is taken), or 0 with an error message on a bad configuration: the order, the
 * backward's workspace.  has_pos: pos is not NULL. */
#define LLATTN_EMBED_ORDER 0
#define LLATTN_EMBED_BACKWARD 1
size_t llattn_embed_bytes(const llattn_embed_cfg* cfg, int32_t has_pos, int32_t which);
int32_t llattn_embed_order(const llattn_embed_cfg* cfg, const void* ids, const void* pos, int32_t tokens, int32_t positions,
                           void* order, size_t order_bytes, void* stream);
int32_t llattn_embed_bwd(const llattn_embed_cfg* cfg, const void* ids, const void* pos, const void* order, const void* dout,
                         void* dW, void* dPos, void* workspace, size_t workspace_bytes, void* stream);

/* ---- the norm over a list of gradients, and clipping -------------------------
 *   norm = sqrt(sum over all elements of g^2),  c = min(1, max_norm / (norm + 1e-6)),  out = c g
 * with squares, sums and products in 64 bits and one rounding to each output's
 * type.  g, out, numel and dtype are host arrays of n entries, read during the
 * call: tensors of numel[i] contiguous elements of dtype[i] at any alignment of
 * whole elements (0 elements: skipped).  A norm that is not finite reaches the
 * gradients: infinity makes c zero (and infinite gradients NaN), NaN makes them
 * all NaN.
 *
 * llattn_grad_norm writes the norm (fp32).  llattn_clip_grads also writes out[i]
 * (out NULL: in place; where c is 1 nothing is written in place); out[i] may be
 * g[i] itself and overlaps nothing else.  With norm_in (a device fp32 value
 * outside of what is written) that is the norm and none is computed (norm NULL
 * then). */
size_t llattn_grad_norm_bytes(int32_t n, const int64_t* numel);
int32_t llattn_grad_norm(int32_t n, const void* const* g, const int64_t* numel, const int32_t* dtype, float* norm,
                         void* workspace, size_t workspace_bytes, void* stream);
int32_t llattn_clip_grads(int32_t n, const void* const* g, void* const* out, const int64_t* numel, const int32_t* dtype,
                          double max_norm, const float* norm_in, float* norm, void* workspace, size_t workspace_bytes,
                          void* stream);

/* ---- gated feed-forward ------------------------------------------------------
 *   a = x W1^T + b1,  u = x W3^T + b3,  h = act(a) u,  y = h W2^T + b2
 * with x [rows][D], W1 and W3 [F][D], W2 [D_out][F], y [rows][D_out], all bf16,
 * biases fp32 or NULL; products summed in fp32, a and u not rounded, h rounded
 * to bf16, which the last product reads; up to 64 rows it is the sum of two bf16
 * values (16 bits), and so are da and du below: infinities of W2 and dy can give
 * NaN there.  act: LLATTN_GATE_SILU a / (1 + exp(-a)) or LLATTN_GATE_GELU
 * a Phi(a).  D, F and D_out are multiples of 8, weights and y contiguous, x of
 * row stride ldx (a multiple of 8, below 2^23); everything 16-byte aligned.
 *
 * Forward: y; with `kept` not NULL (llattn_gated_bytes(cfg, LLATTN_GATED_KEPT)
 * bytes of the caller's) also what the backward reads.  Backward of it, given dy
 * [rows][D_out] contiguous, with p = act(a) and s = act'(a) u:
 *   dh = dy W2,  da = dh s,  du = dh p  (da and du rounded as h is),
 *   dx = da W1 + du W3,  dW1 = da^T x,  dW3 = du^T x,  dW2 = dy^T h,
 *   db1, db3, db2: sums of da, du, dy over the rows (fp32)
 * (any of them NULL; dW1 and dW3 together), dx bf16, dW1 and dW3 of dw_dtype, dW2
 * of dw2_dtype.  Sums run in a fixed order (no atomics). */
#define LLATTN_GATE_SILU 0
#define LLATTN_GATE_GELU 1

typedef struct llattn_gated_cfg {
  int32_t rows, D, F, D_out; /* rows below 2^23 */
  int32_t act;
  int32_t dw_dtype, dw2_dtype; /* LLATTN_F32 or LLATTN_BF16 */
} llattn_gated_cfg;

typedef struct llattn_gated_weights {
  const void *W1, *W3, *W2;
  const float *b1, *b3, *b2;
} llattn_gated_weights;

typedef struct llattn_gated_grads {
  void *dx, *dW1, *dW3, *dW2;
  float *db1, *db3, *db2;
} llattn_gated_grads;

/* Bytes of a buffer (1: none is needed, NULL is taken); 0 with an error message on a bad configuration: workspace of a forward with
 * `kept`, of one without, of the backward; what is kept between them. */
#define LLATTN_GATED_FORWARD 0
#define LLATTN_GATED_ALONE 1
#define LLATTN_GATED_BACKWARD 2
#define LLATTN_GATED_KEPT 3
size_t llattn_gated_bytes(const llattn_gated_cfg* cfg, int32_t which);
int32_t llattn_gated_fwd(const llattn_gated_cfg* cfg, const void* x, int64_t ldx, const llattn_gated_weights* w, void* kept,
                         void* y, void* workspace, size_t workspace_bytes, void* stream);
int32_t llattn_gated_bwd(const llattn_gated_cfg* cfg, const void* x, int64_t ldx, const llattn_gated_weights* w,
                         const void* kept, const void* dy, const llattn_gated_grads* grads, void* workspace,
                         size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LLATTN_LM_H */

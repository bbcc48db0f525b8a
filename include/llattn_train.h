/* The loss and the update of a training step, for the language model around
 * the block: softmax cross entropy over a vocabulary in pieces, and the
 * orthogonalised update of weight matrices.  Same conventions as llattn.h
 * (status codes, llattn_last_error, explicit stream, caller-supplied memory,
 * nothing allocated, no state kept between calls).  No counterpart in the
 * reference beyond the loss itself (reference train.py:354-370). */
#ifndef LLATTN_TRAIN_H
#define LLATTN_TRAIN_H

#include "llattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- softmax cross entropy of h W^T, no logits kept ------------------------
 * l[n][v] = sum_d h[n][d] W[v][d] in fp32 from bf16 h [rows][D], W [V][D] (row
 * strides ldh, ldw in elements, multiples of 8; bases 16-byte aligned; D a
 * multiple of 8, any V, below 2^23 rows).
 *
 * Forward: loss[n] = logsumexp_v l[n] - l[n][t_n] (0 where t_n ==
 * ignore_index, NaN where t_n lies outside [0, V) otherwise), lse2[n] =
 * logsumexp_v l[n] / ln 2 (what the backward reads, and nothing else does),
 * and, with pred non-null, pred[n] = first index of the row's maximum.  With
 * total non-null (one fp32 value): the sum of loss, or with inv non-null too
 * its mean over the rows that count, inv receiving 1 / their number (NaN and 0
 * where there are none).
 *
 * Backward: dl[n][v] = (softmax(l[n])_v - [v == t_n]) * s_n with s_n =
 * grad[n * grad_stride] (grad_stride 0 or 1) * (inv ? *inv : 1), 0 in
 * ignored rows and NaN where t_n is out of range; dh = dl W (bf16 [rows][D],
 * or NULL) and dW = dl^T h (bf16 or fp32 per dw_dtype, [V rounded up to a
 * multiple of 8][D], its rows past V zero, or NULL).  The logits are computed
 * again, `piece` columns of the vocabulary at a time (a multiple of 256, or 0:
 * as many as keep dl, bf16, within 512 MB); dl holds one piece.  Sums run in a fixed order
 * (no atomics). */
typedef struct llattn_head_cfg {
  int32_t rows, V, D;
  int32_t piece;
  int32_t dw_dtype; /* LLATTN_F32 or LLATTN_BF16 */
} llattn_head_cfg;

/* Workspace bytes of llattn_head_fwd (which = 0) and llattn_head_bwd (which =
 * 1); 0 with an error message on sizes that are not supported. */
size_t llattn_head_bytes(const llattn_head_cfg* cfg, int32_t which);
int32_t llattn_head_fwd(const llattn_head_cfg* cfg, const void* h, int64_t ldh, const void* W, int64_t ldw,
                        const int64_t* targets, int64_t ignore_index, float* loss, float* lse2, int32_t* pred,
                        float* total, float* inv, void* workspace, size_t workspace_bytes, void* stream);
int32_t llattn_head_bwd(const llattn_head_cfg* cfg, const void* h, int64_t ldh, const void* W, int64_t ldw,
                        const int64_t* targets, int64_t ignore_index, const float* lse2, const float* grad,
                        int32_t grad_stride, const float* inv, void* dh, void* dW, void* workspace,
                        size_t workspace_bytes, void* stream);

/* ---- orthogonalised matrices and the weight update made of them ------------
 * ns(U): Newton-Schulz iteration towards the orthogonal polar factor of U
 * [rows][cols].  With X = U / (|U|_F + eps), transposed if rows > cols,
 *   A = X X^T,  B = b A + c A A,  X <- a X + B X     (steps times)
 * and transposed back.  Every matrix of the iteration is held as two fp16
 * halves (22 bits of significand) and every product as three products of
 * halves with fp32 accumulation, so results are about as near to the exact ones
 * as fp32 products' are; matrices of at most 16 rows or columns are taken in 64
 * bits (with tiles 0, while |a|^(2 steps) is up to 1e10).  a, b, c, eps and mu count as fp32 holds them.  Fixed
 * order of every sum (no atomics).
 *
 * Matrices come in groups of one shape and type (at most LLATTN_MUON_GROUPS a
 * call, LLATTN_MUON_BATCH matrices, of at most 32768 rows and columns), which
 * share launches whatever their shapes.  Rows are contiguous.
 *
 * llattn_orthogonalize: out[i] = ns(g[i]), g_dtype in, w_dtype out.
 * llattn_muon_update: one optimiser step,
 *   m_out = mu m + (1 - mu) g,  U = nesterov ? (1 - mu) g + mu m_out : m_out,
 *   w_out = keep w - step ns(U)
 * with g in g_dtype, m fp32, w in w_dtype; m_out may be m and w_out may be w
 * (the same arrays), nothing else may overlap.
 *
 * g, m, w, ... are host arrays of device pointers, the groups' matrices in
 * order, read during the call.  a, b, c must keep singular values in [0, 1]
 * below 3.8 and |b s^2 + c s^4| below 15 over the steps (what the halves hold). */
#define LLATTN_MUON_BATCH 128
#define LLATTN_MUON_GROUPS 16

typedef struct llattn_muon_group {
  int32_t batch, rows, cols;
  int32_t g_dtype, w_dtype; /* LLATTN_F32 or LLATTN_BF16 */
  float keep, step;         /* llattn_muon_update */
} llattn_muon_group;

typedef struct llattn_muon_cfg {
  int32_t n_groups;
  int32_t steps, nesterov;
  int32_t tiles; /* of the products: 0: chosen from the sizes, 1: 64 x 64, 2: 64 x 64 in two k groups, 3: 128 x 128,
                    4: 256 x 256 (small matrices in one workgroup each: with 0 only) */
  float a, b, c, eps;
  float mu; /* llattn_muon_update */
} llattn_muon_cfg;

/* Workspace bytes of either call; 0 with an error message on a bad configuration. */
size_t llattn_muon_bytes(const llattn_muon_cfg* cfg, const llattn_muon_group* groups);
int32_t llattn_orthogonalize(const llattn_muon_cfg* cfg, const llattn_muon_group* groups, const void* const* g,
                             void* const* out, void* workspace, size_t workspace_bytes, void* stream);
int32_t llattn_muon_update(const llattn_muon_cfg* cfg, const llattn_muon_group* groups, const void* const* g,
                           const float* const* m, const void* const* w, float* const* m_out, void* const* w_out,
                           void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LLATTN_TRAIN_H */

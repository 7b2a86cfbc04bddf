/*
 * mtffn.h -- C ABI of a gated feed-forward block and of what a training step does with its
 * gradients (libmtgemm.so, beside mtgemm.h and mtlowbit.h, whose conventions hold here too:
 * device pointers, element offsets and strides read in place, work enqueued on `stream`, no
 * allocation, no synchronisation, workspaces sized by the matching query, negative mt_status
 * on error, nothing thrown, every sum in a fixed order).
 *
 * None of these has a counterpart in the reference.  fp32 operands are mt_mat_f32 views with
 * batch 1 unless said otherwise; extents are below 2^31 - 2^16.  An output must not overlap an
 * input unless said otherwise.
 */
#ifndef MTFFN_H
#define MTFFN_H

#include "mtgemm.h"
#include "mtlowbit.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activations, and their formulas: s(a) = 1/(1 + exp(-a)). */
typedef enum mt_activation {
    MT_ACT_SILU = 0,        /* a*s(a) */
    MT_ACT_GELU = 1,        /* a*(1 + erf(a/sqrt 2))/2 */
    MT_ACT_GELU_TANH = 2,   /* a*(1 + tanh(sqrt(2/pi)*(a + 0.044715 a^3)))/2 */
    MT_ACT_RELU = 3,        /* max(a, 0) */
    MT_ACT_SIGMOID = 4      /* s(a) */
} mt_activation;

/* ---- gated feed-forward block ----------------------------------------------------
 * GU = X·Wᵀ + bias with W [2F][in], the gates' rows first;  H = act(GU[:, :F]) * GU[:, F:].
 * GU NULL: not wanted (training keeps it for the backward pass).  bias NULL: none.  No
 * inputs (in = 0): GU is the bias, or zeros.
 * The products are those of mt_linear_forward_f32 and mt_linear_q8.
 * workspace (fp32): a multiple of 4. */
int mt_gated_linear_f32(const mt_mat_f32* X, const mt_mat_f32* W, const float* bias,
                        int64_t bias_stride, int act, const mt_mat_f32* H, const mt_mat_f32* GU,
                        void* workspace, size_t ws_bytes, void* stream);
size_t mt_gated_linear_workspace_f32(const mt_mat_f32* X, const mt_mat_f32* W);
int mt_gated_linear_q8(const mt_rows_q8* X, const mt_rows_q8* W, const float* bias,
                       int64_t bias_stride, int act, const mt_mat_f32* H, const mt_mat_f32* GU,
                       void* workspace, size_t ws_bytes, void* stream);
size_t mt_gated_linear_q8_workspace(const mt_rows_q8* X, const mt_rows_q8* W);
/* The kernel that a call takes (as mt_linear_q8_plan); in fp32: kind 0 straight from
 * memory (tile_rows 16, 32 or 48 on the matrix units, 0 on the vector units), 1 tiles, 2 the product
 * first, then the gate (operands with no unit stride, no inputs). */
typedef struct mt_gate_plan {
    int32_t kind, tile_rows, tile_cols, splits;
    int32_t vector_rows;    /* on the vector units: rows that the kernel is made for, 1, 2, 4, 8
                               or 16; 0: another kernel */
} mt_gate_plan;
int mt_gated_linear_plan_f32(const mt_mat_f32* X, const mt_mat_f32* W, mt_gate_plan* plan);
int mt_gated_linear_q8_plan(int64_t rows, int64_t in_features, int64_t features, mt_q8_plan* plan);

/* H = act(GU[:, :F]) * GU[:, F:] of projections that are there already, and the gradient
 * at them:  dG = dH * U * act'(G),  dU = dH * act(G).  dGU may be the same view as GU.  Of finite
 * operands dG overflows only where the whole product does. */
int mt_gate_f32(const mt_mat_f32* GU, int act, const mt_mat_f32* H, void* stream);
int mt_gate_backward_f32(const mt_mat_f32* dH, const mt_mat_f32* GU, int act,
                         const mt_mat_f32* dGU, void* stream);

/* ... and db = beta*db + the sums of dGU over the rows, the gradient of the projections' bias,
 * from the same pass (mt_linear_backward_f32 then needs no db).  beta 0: db is not read.
 * Eight rows at a time are added up in fp32 and the rest in fp64, so that db is off by no more
 * for many rows than for few.
 * workspace: a multiple of 4. */
int mt_gate_backward_bias_f32(const mt_mat_f32* dH, const mt_mat_f32* GU, int act,
                              const mt_mat_f32* dGU, float* db, int64_t db_stride, float beta,
                              void* workspace, size_t ws_bytes, void* stream);
size_t mt_gate_backward_bias_workspace_f32(int64_t rows, int64_t features);

/* ---- gradients of a whole model ----------------------------------------------------
 * norm = sqrt(sum of the squares of every element of every tensor), held in fp64 until it is
 * rounded to fp32.  Tensors are views of up to three axes (batch, rows, cols), each below 2^42
 * elements, at most 2^20 of them; `grads` is read before the call returns.
 * workspace: a multiple of 8. */
int mt_grad_norm_f32(const mt_mat_f32* grads, int64_t count, float* norm, void* workspace,
                     size_t ws_bytes, void* stream);
/* ... and out[i] = grads[i] * c with c = min(1, max_norm / (norm + eps)), all in fp64 but for
 * the arguments, the product rounded to fp32 once (a NaN among the gradients gives NaN
 * throughout; an infinity 0, and NaN where the gradient is infinite).  out NULL: in place; with
 * c = 1 nothing is written then.  Otherwise out[i] has the shape of grads[i], and may be the
 * same view; but for that no output may overlap another tensor (refused, but for views with
 * gaps between their elements, of which only the first one is looked at).  norm is that before
 * the scaling. */
int mt_clip_grad_norm_f32(const mt_mat_f32* grads, const mt_mat_f32* out, int64_t count,
                          float max_norm, float eps, float* norm, void* workspace, size_t ws_bytes,
                          void* stream);
size_t mt_grad_norm_workspace_f32(int64_t count);

#ifdef __cplusplus
}
#endif

#endif /* MTFFN_H */

/*
 * mtlowbit.h -- C ABI of the operators around a Linear layer whose activations
 * are kept in 8 bits and whose weights are served in 4 (libmtgemm.so, beside
 * mtgemm.h, whose conventions hold here too: device pointers, element offsets
 * and strides read in place, work enqueued on `stream`, no allocation, no
 * synchronisation, workspaces sized by the matching query, negative mt_status
 * on error, nothing thrown, every sum in a fixed order).
 *
 * None of these has a counterpart in the reference, whose tensors are fp32
 * only; their fp32 operands are mt_mat_f32 views with batch 1.
 *
 * Sums and norms are fp32.  Extents are below 2^31 - 2^16, and a product has
 * fewer than 2^23 tiles of 64 x 128 (strides and offsets are 64-bit).  An output must not overlap an input unless said otherwise.
 */
#ifndef MTLOWBIT_H
#define MTLOWBIT_H

#include "mtgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows in 8 bits with one scale each: x[r][c] ~ q[r*row_stride + c] * scale[r].
 * As mt_rms_norm_f32 and mt_quantize_q8_f32 write them, with a = max_c |x[r][c]|:
 *   scale = max(a * (1/127), 2^-126),   q = x * (1/scale) to the nearest (ties
 *   to even), so |q| <= 127 and |x - q*scale| <= (0.5 + 2^-16) * scale.
 * A row that holds an infinity or a NaN has the scale inf or NaN and zero codes
 * wherever x*(1/scale) is none: it reads back as NaN throughout.  A row of no
 * columns has a = 0.
 * Readers take any finite scale and any q, -128 among them. */
typedef struct mt_rows_q8 {
    int8_t* q;
    float* scale;           /* [rows] */
    int64_t rows, cols;
    int64_t row_stride;     /* elements of q, >= cols unless rows <= 1 */
} mt_rows_q8;

/* A weight [n][k] in 4 bits with a scale per `group` (32, 64 or 128) inputs:
 * w[r][c] ~ code(r, c) * scale[r*scale_stride + c/group].  Input 2i of row r is
 * the low half of byte packed[r*row_stride + i], input 2i+1 the high half,
 * two's complement (-8..7).  Rows are 16*ceil(k/32) bytes, the inputs past k in
 * the last 16 being read but not used.  packed and row_stride: multiples of 16;
 * n below 2^26, scale_stride below 2^22 unless n <= 1. */
typedef struct mt_weight_q4 {
    uint8_t* packed;
    float* scale;
    int64_t n, k;
    int64_t row_stride;     /* bytes */
    int64_t scale_stride;   /* elements, >= ceil(k/group) unless n <= 1 */
    int32_t group;
} mt_weight_q4;

/* ---- RMS norm with the residual's addition, rows in 8 bits -----------------
 * h = X (+ R);  rstd[r] = 1/sqrt(sum_c h[r][c]^2 / cols + eps);
 * y[r][c] = (h[r][c] * rstd[r]) * weight[c].
 * R, weight, H, Y, Q, rstd may each be NULL: no addition, a weight of ones, an
 * output that is not wanted.  H may be the same view as X or as R (the residual
 * stream updated in place).  Sums of squares past the fp32 range (|h| near
 * 1e19 and more) are infinite: such a row's y is zero.  A row of no columns has
 * the mean square 0: rstd = 1/sqrt(eps). */
int mt_rms_norm_f32(const mt_mat_f32* X, const mt_mat_f32* R, const float* weight,
                    int64_t weight_stride, float eps, const mt_mat_f32* H, const mt_mat_f32* Y,
                    const mt_rows_q8* Q, float* rstd, void* stream);

/* Its gradients, given dY, the h and rstd of the forward pass, and dH0 (NULL:
 * none), the gradient that arrives at h along the residual stream:
 *   g = dY * weight;  xh = h * rstd;
 *   dH = dH0 + rstd * (g - xh * (sum_c g*xh / cols))   (= dX = dR)
 *   dweight[c] = beta * dweight[c] + sum_r dY[r][c] * xh[r][c].
 * dH or dweight may be NULL.  dH may be the same view as dH0.  Rounding to 8
 * bits passes a gradient through unchanged. */
int mt_rms_norm_backward_f32(const mt_mat_f32* dY, const mt_mat_f32* H, const float* weight,
                             int64_t weight_stride, const float* rstd, const mt_mat_f32* dH0,
                             const mt_mat_f32* dH, float* dweight, int64_t dweight_stride,
                             float beta, void* workspace, size_t ws_bytes, void* stream);
size_t mt_rms_norm_backward_workspace_f32(int64_t rows, int64_t cols);

/* ---- rows kept in 8 bits ---------------------------------------------------- */
int mt_quantize_q8_f32(const mt_mat_f32* X, const mt_rows_q8* Q, void* stream);
int mt_dequantize_q8_f32(const mt_rows_q8* Q, const mt_mat_f32* Y, void* stream);

/* A Linear layer's gradients from an input that was kept in 8 bits (the layout
 * of mt_linear_backward_f32): dX = dY·W, dW = dYᵀ·(scale*q) (+ beta_w·dW_old),
 * db = sum of dY's rows (+ beta_b·db_old).  Any of dX, dW, db may be NULL, and
 * W where dX is.  dW takes dY·scale first, rounded to fp32 (infinite past its
 * range) and to a multiple of 2^-133. */
int mt_linear_backward_q8_f32(const mt_mat_f32* dY, const mt_rows_q8* X, const mt_mat_f32* W,
                              const mt_mat_f32* dX, const mt_mat_f32* dW, float beta_w, float* db,
                              int64_t db_stride, float beta_b, void* workspace, size_t ws_bytes,
                              void* stream);
size_t mt_linear_backward_q8_workspace_f32(int64_t batch_rows, int64_t in_features,
                                           int64_t out_features);

/* ---- Linear over 4-bit weights ----------------------------------------------
 * Codes and scales of a weight: per group, scale = max(max|w| * (1/7), 2^-126),
 * code = w * (1/scale) to the nearest, within -7..7; the inputs that fill up the
 * last 16 bytes are zero.  A group that holds an infinity or a NaN reads back
 * as NaN throughout. */
int mt_quantize_q4_f32(const mt_mat_f32* W, const mt_weight_q4* Q, void* stream);
int mt_dequantize_q4_f32(const mt_weight_q4* Q, const mt_mat_f32* W, void* stream);

/* Y = X·Wᵀ + bias (bias NULL: none), X in fp32 or in 8 bits.  k == 0 writes the bias
 * or zeros.  An fp32 input is taken to the nearest multiple of 2^-133 (which one below
 * 2^-110 need not be); a NaN whose set bits are all in its lower half (a
 * signalling one) counts as an infinity.  Sums are held in fp32, those over 8-bit rows
 * without the row's scale; below 2^-122 they, and with 8-bit rows a group's scale, may
 * be rounded to multiples of 2^-145. */
int mt_linear_q4_f32(const mt_mat_f32* X, const mt_weight_q4* W, const float* bias,
                     int64_t bias_stride, const mt_mat_f32* Y, void* workspace, size_t ws_bytes,
                     void* stream);
int mt_linear_q4_q8(const mt_rows_q8* X, const mt_weight_q4* W, const float* bias,
                    int64_t bias_stride, const mt_mat_f32* Y, void* workspace, size_t ws_bytes,
                    void* stream);
/* Workspace of either call for `rows` rows of X. */
size_t mt_linear_q4_workspace(int64_t rows, int64_t in_features, int64_t out_features);

/* ---- Linear over 8-bit weights -------------------------------------------------
 * Y = X·Wᵀ + bias, both operands in 8 bits: W's rows are the output channels, a scale
 * each (mt_quantize_q8_f32 of the weight gives them):
 *   y[m][n] = (sum_k X.q[m][k]·W.q[n][k]) * X.scale[m] * W.scale[n] + bias[n].
 * The sum is exact, whatever its length, and rounded to fp32 once; so is its product with one
 * scale, and y.  No finite scales overflow where y does not.  Rows may lie at any
 * address; of many rows of X (mt_linear_q8_plan: tiles), an operand whose rows do not start on
 * multiples of 16 bytes is first copied to the workspace. */
int mt_linear_q8(const mt_rows_q8* X, const mt_rows_q8* W, const float* bias, int64_t bias_stride,
                 const mt_mat_f32* Y, void* workspace, size_t ws_bytes, void* stream);
size_t mt_linear_q8_workspace(const mt_rows_q8* X, const mt_rows_q8* W);

/* ---- diagnostics ---------------------------------------------------------------
 * Which kernel a product's call takes, by its sizes, for tests and benchmarks (as
 * mt_last_config, but nothing runs): of the 4-bit product, and of dW. */
typedef struct mt_lowbit_plan {
    int32_t tile_rows;      /* 64 or 128, by twice as many columns; 0: the few-rows kernel */
    int32_t splits;         /* of the summed axis, added up by a launch of their own */
    int32_t column_blocks;  /* of 16 columns, a workgroup of the few-rows kernel; 0 with tiles */
} mt_lowbit_plan;
/* Of a product with 8-bit weights: 64x128, 128x128, 128x256 or 256x256; 0: a kernel without
 * tiles. */
typedef struct mt_q8_plan {
    int32_t tile_rows, tile_cols;
    int32_t splits;
    int32_t row_blocks, column_blocks;   /* without tiles: of 16 rows and of 16 columns (gated:
                                            half of them gates), a workgroup; 0 with tiles */
} mt_q8_plan;
int mt_linear_q4_plan(int64_t rows, int64_t in_features, int64_t out_features, int group,
                      int x_in_8_bits, mt_lowbit_plan* plan);
int mt_linear_q8_plan(int64_t rows, int64_t in_features, int64_t out_features, mt_q8_plan* plan);
int mt_linear_backward_q8_plan(int64_t batch_rows, int64_t in_features, int64_t out_features,
                               mt_lowbit_plan* plan);

#ifdef __cplusplus
}
#endif

#endif /* MTLOWBIT_H */

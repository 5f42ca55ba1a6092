/*
 * gnn_train.h -- the training operators of libgnnagg.so that stand around the aggregation path: RMS norm with the
 * residual's addition, dense products in 8-bit floating point, and an AdamW step over many tensors.  Written for AMD
 * MI355X (gfx950).  A second header with a version of its own: gnn_agg.h and its version stay as they are.
 *
 * Conventions are gnn_agg.h's: every pointer is a DEVICE pointer unless its comment says "host", `stream` is a
 * hipStream_t as void*, every entry point only enqueues work on it (no allocation, no synchronisation, no memset: all
 * of them can be recorded into a HIP graph), returns GNNAGG_OK or an error code whose text gnnagg_last_error() gives,
 * and is deterministic (no floating-point atomics).  The current HIP device has to be the pointers' device.
 *
 * THE 8-BIT FORMAT.  Values are e4m3 codes (OCP, largest 448, no infinity) in blocks of 128; a block's scale is a power
 * of two kept as one byte, 2^(byte - 127) (e8m0): the smallest exponent e in [-126, 120] with max|x| * 2^-e <= 448 over
 * the block's finite values.  code = e4m3 nearest to x * 2^-e (ties to even; the product is exact, so a code depends on
 * nothing but x and its block); an infinity or NaN becomes the NaN code and does not touch the scale.
 *   rows     codes [rows][pitch] with pitch = width rounded up to 128, the padding zero; scales [rows][pitch / 128]
 *   weights  of a matrix W [K, N]: codes by output [N][K rounded up to 128] and, for the input gradient, codes by input
 *            [K][N rounded up to 128], both with zero padding and both with the scales of W's 128 x 128 blocks,
 *            [ceil(K / 128)][ceil(N / 128)]
 *
 * `dtype` arguments: GNNAGG_F32 or GNNAGG_BF16.  Strides are in elements.
 */
#ifndef GNN_TRAIN_H
#define GNN_TRAIN_H

#include "gnn_agg.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GNNAGG_F32 0
#define GNNAGG_BF16 1

/* Raised whenever a prototype of this header changes, comes or goes; bindings compare it with
 * gnnagg_train_abi_version() before the first call. */
#define GNNAGG_TRAIN_ABI_VERSION 1
int gnnagg_train_abi_version(void);

/* ---------------------------------------------------------------------------------
 * RMS norm with the residual's addition, rows of `width` <= 16384 values:
 *   h = x + residual (rounded to dtype; h = x where residual is NULL)
 *   y = h / sqrt(mean(h^2) + eps) * weight, then max(y, 0) where relu != 0
 * The mean square is summed in 64 bits, the rest is fp32.  In a row with an infinity the inverse root is zero: its finite
 * values give zero, its infinite ones NaN.  A NaN makes its whole row NaN.
 *   x, residual (or NULL), h (written where residual is given, NULL otherwise), y: dtype, row strides of their own
 *   weight: [width], weight_dtype GNNAGG_F32 or dtype
 * ------------------------------------------------------------------------------- */
int gnnagg_rms_norm(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight,
                    int weight_dtype, double eps, int relu, void *h, int64_t h_stride, void *y, int64_t y_stride,
                    int64_t rows, int64_t width, int dtype, void *stream);

/* The same with y leaving in the 8-bit format's rows (taken from the fp32 value of y, no rounding to dtype between). */
int gnnagg_rms_norm_fp8(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                        const void *weight, int weight_dtype, double eps, int relu, void *h, int64_t h_stride,
                        uint8_t *codes, uint8_t *scales, int64_t rows, int64_t width, int dtype, void *stream);

/* Gradient.  grad_y and grad_h (the gradient of the residual stream; NULL: none): dtype; h: what the forward normalised;
 * grad_x: dtype, the gradient of x and of the residual alike; grad_weight: [width] fp32.
 * workspace: gnnagg_rms_norm_backward_workspace_bytes (checked), any contents. */
int64_t gnnagg_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width);
int gnnagg_rms_norm_backward(const void *grad_y, int64_t grad_y_stride, const void *grad_h,
                             int64_t grad_h_stride, const void *h, int64_t h_stride, const void *weight,
                             int weight_dtype, double eps, int relu, void *grad_x, int64_t grad_x_stride,
                             float *grad_weight, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t width,
                             int dtype, void *stream);

/* ---------------------------------------------------------------------------------
 * Dense products in the 8-bit format.
 * ------------------------------------------------------------------------------- */

/* x [rows, width] (dtype, row stride x_stride) -> codes, scales of the format's rows. */
int gnnagg_fp8_quantize_rows(const void *x, int64_t x_stride, uint8_t *codes, uint8_t *scales, int64_t rows,
                             int64_t width, int dtype, void *stream);

/* w [K, N] (dtype, row stride w_stride) -> codes_by_output [N][K padded], codes_by_input [K][N padded] (either may be
 * NULL), scales [ceil(K / 128)][ceil(N / 128)]. */
int gnnagg_fp8_quantize_weight(const void *w, int64_t w_stride, uint8_t *codes_by_output, uint8_t *codes_by_input,
                               uint8_t *scales, int64_t k, int64_t n, int dtype, void *stream);

/* out[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]), accumulated in fp32, stored as out_dtype.  GNNAGG_F32: products exact, for
 * scales in [2^-124, 2^119] (below, the smallest codes are rounded to bf16's subnormals; 2^128 is infinite).  GNNAGG_BF16: of the
 * products of eight neighbouring codes each is cut to a multiple of 2^-13 of the largest one's power of two (the 8-bit
 * matrix instruction's way), at any scale.
 *   x codes [rows][k padded] with scales [rows][k padded / 128]; w codes [n][k padded] whose block (kb, nb) has the
 *   scale w_scales[kb * scale_k_stride + nb * scale_n_stride]; bias fp32 [n] or NULL; out row stride out_stride.
 * Codes and padding are read whole: 16-byte aligned, k padded to a multiple of 128.  The forward product takes the codes
 * by output, the input gradient the codes by input with the two scale strides exchanged. */
int gnnagg_fp8_product(const uint8_t *x, const uint8_t *x_scales, const uint8_t *w, const uint8_t *w_scales,
                       int64_t scale_k_stride, int64_t scale_n_stride, const float *bias, void *out, int64_t out_stride,
                       int out_dtype, int64_t rows, int64_t k, int64_t n, void *stream);

/* grad_w[k, n] = sum_m x[m, k] * bf16(g[m, n]) in fp32 (x: the format's rows; a code times a scale in [2^-124, 2^119] is a
 * bf16 value, so x enters exactly; outside as for the fp32 product) and, where grad_bias is not NULL, grad_bias[n] = sum_m g[m, n] in fp32.
 * g: g_dtype, row stride g_stride.  grad_w fp32 [k][n].  workspace: gnnagg_fp8_weight_gradient_workspace_bytes (checked),
 * any contents. */
int64_t gnnagg_fp8_weight_gradient_workspace_bytes(int64_t rows, int64_t k, int64_t n);
int gnnagg_fp8_weight_gradient(const uint8_t *x, const uint8_t *x_scales, const void *g, int64_t g_stride, int g_dtype,
                               float *grad_w, float *grad_bias, void *workspace, int64_t workspace_bytes, int64_t rows,
                               int64_t k, int64_t n, void *stream);

/* ---------------------------------------------------------------------------------
 * AdamW (decoupled weight decay) over `count` tensors.  For each: t = ++steps[i];
 *   m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
 * `tensors`: HOST array, read before the call returns.  n elements each, contiguous; n == 0 is skipped (its step still
 * counts).  param / grad: param_dtype / grad_dtype; with GNNAGG_BF16 parameters `master` is the fp32 value that is
 * updated and param receives it rounded; with fp32 parameters master is NULL.
 *   state_bits 32: exp_avg = m, exp_avg_sq = v, fp32; the scale pointers NULL
 *   state_bits 8:  exp_avg = m, exp_avg_sq = sqrt(v) as codes of the 8-bit format, blocks of 128 elements from the
 *     tensor's start, scales [ceil(n / 128)].  m is rounded to nearest, sqrt(v) to one of its two neighbours with the odds
 *     of the distance (at beta2 = 0.999 a step moves sqrt(v) by far less than half a code, and rounding to nearest would
 *     hold it still); a v above zero never becomes zero.  The 20 random bits of element j of tensor i at step t are a hash
 *     of (seed, first + i, t, j): equal calls give equal results.  `first`: the number of the first tensor, for callers
 *     that split a list over several calls.
 * steps: int32 [count] on the device, the number of steps taken so far, raised by one here: a captured call counts its
 * replays.  lr_tensor: fp32 scalar on the device that is read instead of lr, or NULL.  No memory that is written may
 * overlap any other that is written or read here (not checked at this level).
 * ------------------------------------------------------------------------------- */
typedef struct gnnagg_adamw_tensor {
    void *param;
    const void *grad;
    void *exp_avg;
    void *exp_avg_sq;
    uint8_t *exp_avg_scales;
    uint8_t *exp_avg_sq_scales;
    float *master;
    int64_t n;
} gnnagg_adamw_tensor;

int gnnagg_adamw_step(const gnnagg_adamw_tensor *tensors, int64_t count, int32_t *steps, int param_dtype,
                      int grad_dtype, int state_bits, double lr, const float *lr_tensor, double beta1, double beta2,
                      double eps, double weight_decay, uint32_t seed, int64_t first, void *stream);

#ifdef __cplusplus
}
#endif

#endif

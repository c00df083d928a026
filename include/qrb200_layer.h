/* qrb200 -- layer operators, C ABI: what is done with a factor Q once it is a weight.  A root-mean-square norm
 * commutes with an orthogonal Q (the norm of a row does not change), so activations can be
 * rotated by Q, normed, held in 8 bits and multiplied.  No counterpart in the reference.
 *
 * All pointers are device pointers; rows of a matrix are `ld` elements apart (any ld that keeps
 * rows apart on outputs; inputs may overlap or repeat, ld = 0 included, except matrix-product
 * operands) and contiguous inside; bases and strides need no alignment but their elements'.  A
 * workspace may start at any byte: the queried sizes allow for that.  Everything is
 * enqueued on `stream`; nothing is synchronised.  Empty sizes are a successful no-op
 * (but rows of no elements have their scale written).
 *
 * Status codes, element types and the conventions of qrb200.h; nothing here depends on PyTorch or
 * on the CUDA headers. */
#ifndef QRB200_LAYER_H
#define QRB200_LAYER_H

#include "qrb200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* a further element type: e4m3 with a scale per row, q * scale[row] is the value (largest q 448,
 * no infinity) */
#define QRB200_E4M3 3

/* Root-mean-square norm of rows of `dim` elements, with the residual's addition:
 *   h = x + residual  (rounded to the stream's type; h = x without a residual)
 *   y = h * (mean(h^2) + eps)^-1/2 * weight
 *   x        [rows][dim], `dtype` (F32, BF16, F16)
 *   weight   [dim], `dtype` or F32, or NULL for ones
 *   residual [rows][dim], `stream_dtype` (= `dtype`, or F32), or NULL
 *   y        [rows][dim] contiguous; out_dtype = `dtype`, or E4M3: then scale[rows] is written too,
 *            scale = max(max |y| / 448, 2^-126) of the row, y = e4m3(y / scale), in float32 as
 *            y (1 / scale): beside the middle between two codes either may be taken
 *   h        [rows][dim] contiguous, `stream_dtype`; may be `residual` itself (in place, ldr = dim);
 *            not written (may be NULL) without a residual
 * A NaN in a row makes its y (and scale) NaN. */
int qrb200_rms_norm(const void* x, int64_t ldx, const void* weight, int32_t weight_dtype,
                    const void* residual, int64_t ldr, int32_t stream_dtype, void* y,
                    float* scale, void* h, int64_t rows, int64_t dim, float eps, int32_t dtype,
                    int32_t out_dtype, void* stream);

/* Rows of x [rows][dim] in 8 bits with a scale each, by the rule of qrb200_rms_norm (to lay out
 * weights once: one scale per output feature). */
int qrb200_quantize_rows(const void* x, int64_t ldx, void* q, float* scale, int64_t rows,
                         int64_t dim, int32_t dtype, void* stream);

/* Gradients of qrb200_rms_norm.  dy = gradient of y, dh = gradient of h (NULL: zero), h as the
 * forward pass left it (x without a residual).  With g = dy * weight, r = (mean(h^2)+eps)^-1/2:
 *   dx = dresidual = dh + r g - (r^3 mean(g h)) h,    dweight = sum over rows of dy h r
 *   dy, dx   `dtype`;  h, dh, dresidual `stream_dtype`;  dweight in the weight's type
 * dx, dresidual and dweight are contiguous and may each be NULL; dresidual equals dx, so it is only
 * needed where stream_dtype differs.  The weight's gradient is added up in a fixed order: the same
 * inputs give the same bits.  `workspace` (NULL: allocated stream-ordered) is needed for dweight. */
int qrb200_rms_norm_backward_workspace_bytes(int64_t rows, int64_t dim, int32_t dtype,
                                             int32_t stream_dtype, size_t* bytes);
int qrb200_rms_norm_backward(const void* dy, int64_t lddy, const void* h, int64_t ldh,
                             const void* dh, int64_t lddh, const void* weight,
                             int32_t weight_dtype, void* dx, void* dresidual, void* dweight,
                             int64_t rows, int64_t dim, float eps, int32_t dtype,
                             int32_t stream_dtype, void* workspace, size_t workspace_bytes,
                             void* stream);

/* activations of qrb200_linear */
#define QRB200_ACT_NONE 0
#define QRB200_ACT_RELU 1
#define QRB200_ACT_GELU 2      /* z Phi(z) */
#define QRB200_ACT_GELU_TANH 3 /* its tanh approximation */
#define QRB200_ACT_SILU 4      /* z / (1 + exp(-z)) */

/* Matrix product with its epilogue:
 *   y = act(x_scale_i w_scale_j sum_k x_ik w_jk + bias_j) + residual_ij
 *   x        [m][k], w [n][k], `dtype` BF16, F16 or E4M3; w_transposed != 0: w is stored [k][n]
 *            (not for E4M3)
 *   x_scale  [m], w_scale [n], float32, or NULL for ones; for E4M3 only
 *   bias     [n], residual [m][n], y [m][n]: `out_dtype` (= `dtype`; BF16 or F16 for E4M3);
 *            residual may be y itself (in place)
 *   slope    [m][n] contiguous, or NULL: act'(z) for qrb200_linear_backward as
 *            round(2^15 (t + 3/8)) with act' = t |t|, 65535 for NaN; not for E4M3
 * m and n up to 8388480 (128 * 65535), k up to 2^31 - 65537.  Sums are float32; y is rounded once.
 * `workspace` (NULL: allocated stream-ordered) holds aligned copies of operands whose rows do not
 * all start on 16 bytes; none is needed otherwise. */
int qrb200_linear_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                  int32_t w_transposed, int64_t m, int64_t n, int64_t k,
                                  int32_t dtype, size_t* bytes);
int qrb200_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t w_transposed,
                  const float* x_scale, const float* w_scale, const void* bias,
                  const void* residual, int64_t ldr, void* y, int64_t ldy, uint16_t* slope,
                  int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t out_dtype,
                  int32_t activation, void* workspace, size_t workspace_bytes, void* stream);

/* Gradients of qrb200_linear (BF16, F16), dz = dy * slope (slope NULL: dz = dy):
 *   dx [m][k] = dz w,   dw [n][k] = dz^T x,   dbias [n] = sum over rows of dz
 * contiguous, in `dtype`, each may be NULL.  dz is rounded to `dtype` for the two products and kept
 * in float32 for dbias.  The residual's gradient is dy itself.  Fixed summation order. */
int qrb200_linear_backward_workspace_bytes(const void* dy, int64_t lddy, int32_t has_slope,
                                           const void* x, int64_t ldx, const void* w,
                                           int64_t ldw, int32_t w_transposed, int32_t want_dx,
                                           int32_t want_dw, int32_t want_dbias, int64_t m,
                                           int64_t n, int64_t k, size_t* bytes);
int qrb200_linear_backward(const void* dy, int64_t lddy, const uint16_t* slope, const void* x,
                           int64_t ldx, const void* w, int64_t ldw, int32_t w_transposed,
                           void* dx, void* dw, void* dbias, int64_t m, int64_t n, int64_t k,
                           int32_t dtype, void* workspace, size_t workspace_bytes, void* stream);

/* *timed_out = 1 if a bounded in-kernel wait of a layer operator has run out on the current device
 * since the last call (never expected; the outputs it concerned are NaN).  Waits for all work of the
 * device, on any stream; not while one of its streams is being captured. */
int qrb200_layer_status(int32_t* timed_out);

#ifdef __cplusplus
}
#endif

#endif /* QRB200_LAYER_H */

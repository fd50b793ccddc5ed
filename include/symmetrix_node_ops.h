/*
 * symmetrix_node_ops.h -- C ABI of the node operators (libsymmetrix_mi355x.so):
 * what a learned block over an evaluator's atoms is made of, forward and
 * backward, for training it and for serving it.  The reference has no
 * counterpart.
 *
 *   species embedding     out[t] = scale * table[types[t]], and its gradient
 *   residual norm         y = x + a * sigmoid(g) * post * d / rms(d),
 *                         h = next * y / rms(y), and their gradients
 *   8-bit block product   y = x W^T with E4M3 operands, a scale for each block of
 *                         128 values along the summed axis
 *
 * Conventions are those of symmetrix_mi355x.h (0 or a negative SMX_ERR_* code, no
 * exceptions, smx_last_error() for the message), with these:
 *   - every pointer is a device pointer; every call enqueues on `stream` (a
 *     hipStream_t; NULL: the default stream) of the current device, keeps no
 *     argument and does not wait, so a call may be captured into a HIP graph;
 *   - nothing is allocated: a call that needs room between its kernels takes a
 *     workspace of the size its _workspace function gives (16-byte aligned, the
 *     caller's again when the enqueued work is done);
 *   - row arrays are [rows][channels] with unit stride along the channels and
 *     any stride >= channels (in elements) between rows; outputs must not
 *     overlap inputs unless the comment says so;
 *   - values are SMX_DTYPE_* (one type for all row arrays of a call); sums, norms and
 *     products are held in FP32 and rounded once, to nearest even, when they are
 *     stored;
 *   - results do not depend on the order in which workgroups run.
 */
#ifndef SYMMETRIX_NODE_OPS_H
#define SYMMETRIX_NODE_OPS_H

#include <stdint.h>

#include "symmetrix_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { SMX_DTYPE_F32 = 0, SMX_DTYPE_BF16 = 1, SMX_DTYPE_F16 = 2 };

/* ---- species embedding ---- */

/* out[t][c] = scale * table[types[t]][c].  A type outside [0, num_types) is no
 * species (a masked or padding atom): its row is zero.  types: int32, or int64 when
 * types_are_64bit.  Up to 2^31 - 65536 tokens and types. */
SMX_API int32_t smx_embed(const void* types, int32_t types_are_64bit, int64_t tokens, const void* table,
                          int64_t table_stride, int64_t num_types, int64_t channels, int32_t dtype, float scale,
                          void* out, int64_t out_stride, void* stream);
/* out[v][c] = scale * sum over the t with types[t] == v of grad[t][c], every row
 * of out written (zeros for a type without atoms).  Each type's rows are summed
 * in FP32 and a fixed order: the same call gives the same bits. */
SMX_API int64_t smx_embed_gradient_workspace(int64_t tokens, int64_t num_types, int64_t channels);
SMX_API int32_t smx_embed_gradient(const void* types, int32_t types_are_64bit, int64_t tokens, const void* grad,
                                   int64_t grad_stride, int64_t num_types, int64_t channels, int32_t dtype,
                                   float scale, void* out, int64_t out_stride, void* workspace,
                                   int64_t workspace_bytes, void* stream);

/* ---- residual norm ---- */

/* How the gate logits are given: not at all (a gate of one), one for each
 * value ([rows][channels], gate_stride between rows), for each channel
 * ([channels]), or for each row ([rows], gate_stride between them). */
enum { SMX_GATE_NONE = 0, SMX_GATE_FULL = 1, SMX_GATE_CHANNEL = 2, SMX_GATE_ROW = 3 };

/* y = x + scale * sigmoid(gate) * post * d * r1,  r1 = 1 / sqrt(mean(d^2) + eps)
 * h = next * y * r2,                              r2 = 1 / sqrt(mean(y^2) + eps)
 * (means over a row's channels; h is formed from y before it is rounded).
 * post, scale and next are FP32 [channels].  d NULL: y = x, and post, gate and
 * scale are not read.  scale NULL: ones.  y NULL: not written.  next NULL: no h.
 * y may be x.  With h_scales, h is written as 8-bit blocks (below) instead of
 * `dtype`: h the values [rows][smx_block_stride(channels)] and h_scales
 * [rows][smx_block_scale_stride(channels)].  channels <= 16384.  The sigmoid, and one minus it in the gradients, come
 * from the hardware exponential of a logit's magnitude: within 2^-20 of themselves in FP32 rows, whatever the
 * logit (below FP32's normal numbers, from magnitudes of 87 on, zero), and |logit| 2^-24 more in 16-bit rows. */
typedef struct SmxResidualNormArgs {
    uint32_t struct_size;
    int32_t dtype;
    int64_t rows;
    int64_t channels;
    const void* x;
    int64_t x_stride;
    const void* d;
    int64_t d_stride;
    const void* gate;
    int64_t gate_stride;
    int32_t gate_kind;
    float eps;
    const float* post;
    const float* scale;
    const float* next;
    void* y;
    int64_t y_stride;
    void* h;
    int64_t h_stride; /* ignored with h_scales */
    uint8_t* h_scales;
} SmxResidualNormArgs;
SMX_API int32_t smx_residual_norm(const SmxResidualNormArgs* args, void* stream);

/* The gradients with respect to every input, from the inputs alone (nothing
 * of the forward call is kept): of a loss whose gradients with respect to y and h
 * are grad_y (NULL: zero) and grad_h (NULL: zero; needs next).  Each output may be NULL
 * (not formed).  dx, dd and dgate (of the gate's shape) are `dtype`; dpost, dscale and dnext are FP32
 * [channels].  Sums over the rows have a fixed order.  dx may be grad_y. */
typedef struct SmxResidualNormGradientArgs {
    SmxResidualNormArgs forward; /* y, h and h_scales are not used */
    const void* grad_y;
    int64_t grad_y_stride;
    const void* grad_h;
    int64_t grad_h_stride;
    void* dx;
    int64_t dx_stride;
    void* dd;
    int64_t dd_stride;
    void* dgate;
    int64_t dgate_stride;
    float* dpost;
    float* dscale;
    float* dnext;
    void* workspace;
    int64_t workspace_bytes;
} SmxResidualNormGradientArgs;
SMX_API int64_t smx_residual_norm_gradient_workspace(int64_t rows, int64_t channels);
SMX_API int32_t smx_residual_norm_gradient(const SmxResidualNormGradientArgs* args, void* stream);

/* ---- 8-bit block product ---- */

/* A matrix [rows][cols] in 8-bit blocks: E4M3 values [rows][smx_block_stride(cols)]
 * (cols rounded up to 128, the rest zeros) and one E8M0 scale byte b, the scale
 * 2^(b-127), for each block of 128 values of a row: [rows][smx_block_scale_stride(cols)]
 * (the number of blocks rounded up to 4, the rest zeros).  A block's scale is the
 * least power of two >= 2^-127 that brings its largest finite magnitude to 448 or less; values
 * round to nearest even; an infinity or NaN is stored as NaN.  Both arrays must be
 * 16-byte aligned. */
SMX_API int64_t smx_block_stride(int64_t cols);
SMX_API int64_t smx_block_scale_stride(int64_t cols);
/* x [rows][cols] in blocks along its rows (values, scales) and/or the blocks of
 * its transpose, [cols][rows] in blocks along the rows of x (values_t, scales_t);
 * either pair may be NULL. */
SMX_API int32_t smx_block_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols,
                                   uint8_t* values, uint8_t* scales, uint8_t* values_t, uint8_t* scales_t,
                                   void* stream);
/* out[i][j] = sum over k of a[i][k] b[j][k], a [m][k] and b [n][k] in 8-bit blocks, k < 2^23 - 127.
 * FP32 outputs, and 16-bit ones of up to 256 terms, are FP32 sums of the operands' values as bf16 numbers,
 * which hold them exactly from 2^-126 on, round them to multiples of 2^-133 below, and have infinity for the one value
 * that is beyond FP32 (2^128, to which the largest FP32 numbers round).  16-bit outputs of more than
 * 256 terms come from the 8-bit matrix instruction, which takes every value as it is but aligns eight products to the
 * largest of them and drops what lies 2^-13 below it: up to 7 x 2^-13 of the largest of each eight.  In sums of many
 * terms of one size that is about 2^-16 of an output's norm, below the outputs' own rounding (2^-9 or 2^-12); where
 * single products stand far above the others it may be up to 2^-10 of those, which float16 is finer than and which stays
 * when they cancel: FP32 outputs have neither.  An infinity or NaN in a row of an operand makes that row of products NaN,
 * and no other. */
SMX_API int64_t smx_block_product_workspace(int64_t m, int64_t n, int64_t k);
SMX_API int32_t smx_block_product(const uint8_t* a_values, const uint8_t* a_scales, const uint8_t* b_values,
                                  const uint8_t* b_scales, int64_t m, int64_t n, int64_t k, int32_t dtype, void* out,
                                  int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream);
/* The same with a = x [m][k] of `dtype`, brought to blocks within the call;
 * out is out_dtype. */
SMX_API int64_t smx_block_linear_workspace(int64_t m, int64_t n, int64_t k);
SMX_API int32_t smx_block_linear(const void* x, int64_t x_stride, int32_t dtype, const uint8_t* w_values,
                                 const uint8_t* w_scales, int64_t m, int64_t n, int64_t k, int32_t out_dtype,
                                 void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes,
                                 void* stream);

/* ---- rows by kind ---- */

/* A plan of `rows` rows by their kind, types[t] in [0, num_types) (int32, or int64 when types_are_64bit); a row of another
 * type is masked.  The plan is device memory (16-byte aligned, smx_group_plan_bytes of it), an input of the products below for
 * the same rows and num_types.  What it is of is known to the device alone: with a plan of others the products return SMX_OK and
 * write nothing, so an output keeps what it held.  As int32 the plan holds from byte 16 on the offsets, num_types + 1 of them (of
 * the sorted rows of type z the first is offsets[z] and the one past the last offsets[z + 1]), and from byte
 * smx_group_plan_order on the rows in order: by type, of one type as they come, the masked ones last.  Up to 2^30 rows and
 * 4,096 types. */
SMX_API int64_t smx_group_plan_bytes(int64_t rows, int64_t num_types);
SMX_API int64_t smx_group_plan_order(int64_t num_types);
SMX_API int64_t smx_group_rows_workspace(int64_t rows, int64_t num_types);
SMX_API int32_t smx_group_rows(const void* types, int32_t types_are_64bit, int64_t rows, int64_t num_types, void* plan,
                               int64_t plan_bytes, void* workspace, int64_t workspace_bytes, void* stream);

/* out[t] = w[z] x[t] with z the type of row t and w [num_types][outputs][inputs] (w_stride between rows, w_type_stride
 * between types, in values); the rows of masked t are zeros.  Values are `dtype`, out is out_dtype: that or FP32.  Products of FP32
 * values are formed of three bf16 parts of each, to FP32's precision (2^-24 of a product; parts are multiples of 2^-133, so a
 * value below 2^-110 is off by up to 2^-134).  An infinity or NaN makes the outputs infinite or NaN that it is a term of, and no
 * others.  inputs, outputs <= 2^24. */
SMX_API int32_t smx_grouped_linear(const void* x, int64_t x_stride, int32_t dtype, const void* w, int64_t w_stride,
                                   int64_t w_type_stride, const void* plan, int64_t rows, int64_t num_types, int64_t inputs,
                                   int64_t outputs, int32_t out_dtype, void* out, int64_t out_stride, void* stream);
/* Its gradients from that of out, grad [rows][outputs]: dx[t] = w[z]^T grad[t], zeros for masked t, */
SMX_API int32_t smx_grouped_linear_by_rows(const void* grad, int64_t grad_stride, int32_t dtype, const void* w, int64_t w_stride,
                                           int64_t w_type_stride, const void* plan, int64_t rows, int64_t num_types,
                                           int64_t inputs, int64_t outputs, int32_t out_dtype, void* dx, int64_t dx_stride,
                                           void* stream);
/* and dw[z] = the sum over rows of type z of grad[t] x[t]^T, every matrix of dw written (zeros for a type without rows), summed
 * in a fixed order. */
SMX_API int64_t smx_grouped_linear_by_weights_workspace(int64_t rows, int64_t num_types, int64_t inputs, int64_t outputs);
SMX_API int32_t smx_grouped_linear_by_weights(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, int32_t dtype,
                                              const void* plan, int64_t rows, int64_t num_types, int64_t inputs,
                                              int64_t outputs, int32_t out_dtype, void* dw, int64_t dw_stride,
                                              int64_t dw_type_stride, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- gradients' norm and clipping ---- */

/* norm = scale * sqrt(sum of the squares of all values) of num_tensors tensors of counts[i] values of type dtypes[i], packed.
 * tensors, counts and dtypes are host arrays, read within the call; tensors' values, norm and the workspace are on the device.
 * Squares and sums are FP64 and have a fixed order, so no FP32 value is too large for its square, and norm is rounded once.
 * scale (of gradients whose loss was scaled, 1 / the loss's) is positive and finite.  Up to 98,304 tensors. */
SMX_API int64_t smx_gradient_norm_workspace(void);
SMX_API int32_t smx_gradient_norm(const void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t num_tensors,
                                  float scale, float* norm, void* workspace, int64_t workspace_bytes, void* stream);
/* The same, and out[i] = tensors[i] * scale * min(1, max_norm / norm) in out_dtypes[i]: out[i] may be tensors[i] where its type
 * is the same; outputs overlap nothing else.  The factor is from the norm in FP64 and rounded to FP32's 24 bits
 * whatever its size, and an output is rounded once more, and to its type; a factor of one changes no value.  A norm that is infinite
 * makes every finite value zero and the others NaN (a max_norm that is infinite too clips nothing), one that is NaN makes all NaN: look
 * at norm. */
SMX_API int32_t smx_clip_gradients(const void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t num_tensors,
                                   float max_norm, float scale, void* const* out, const int32_t* out_dtypes, float* norm,
                                   void* workspace, int64_t workspace_bytes, void* stream);

/* ---- products in 8-bit integers ---- */

/* A matrix [rows][cols] in 8-bit integers: values [rows][smx_integer_stride(cols)] (cols rounded up to 128, the rest zeros; 16-byte
 * aligned) and an FP32 scale for each row.  A row's scale is the FP32 product of its largest magnitude and the
 * FP32 number next to 1/127 (0x1.020408p-7), at least 2^-126, and a value the whole number nearest to the exact quotient by the
 * scale, ties to even.  A row with an infinity or NaN has the scale NaN and zeros. */
SMX_API int64_t smx_integer_stride(int64_t cols);
SMX_API int32_t smx_integer_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, int8_t* values,
                                     float* scales, void* stream);
/* out[i][j] = a_scales[i] b_scales[j] sum over k of a[i][k] b[j][k], a [m][k] and b [n][k] as above, k <= 2^17: the sum is exact and
 * is rounded when it becomes FP32, at either scale (so that a product that is a number of FP32 is one), and to `dtype`. */
SMX_API int32_t smx_integer_product(const int8_t* a_values, const float* a_scales, const int8_t* b_values, const float* b_scales,
                                    int64_t m, int64_t n, int64_t k, int32_t dtype, void* out, int64_t out_stride, void* stream);
/* The same with a = x [m][k] of `dtype`, brought to integers within the call; out is out_dtype. */
SMX_API int64_t smx_integer_linear_workspace(int64_t m, int64_t n, int64_t k);
SMX_API int32_t smx_integer_linear(const void* x, int64_t x_stride, int32_t dtype, const int8_t* w_values, const float* w_scales,
                                   int64_t m, int64_t n, int64_t k, int32_t out_dtype, void* out, int64_t out_stride,
                                   void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SYMMETRIX_NODE_OPS_H */

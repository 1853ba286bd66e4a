/*
 * C-ABI of the dense operators around deformable attention in an encoder or
 * decoder layer: the linear layer with its epilogue and gradients, its 8-bit
 * input checkpoint, the gated layer, linear on 8-bit integers, layer norm with its gradients, dropout, and the sum of a block
 * with the residual stream and the norm after it. Part of `libmuspace_msda.so`,
 * MI355X (gfx950).
 *
 * Tensors are device pointers, dense, row-major, all of one type: float32 (0),
 * float16 (1) or bfloat16 (2), unless noted. Products and statistics are summed
 * in float32, in a fixed order; every result is rounded once, to its type. float32
 * products of many rows read their operands to an absolute 2^-134 (magnitudes under
 * 2^-109 keep fewer than float32's 24 bits). Any
 * sizes and any alignment of the type are allowed; rows of whole 16-byte pieces
 * on 16-byte boundaries are the fast case.
 *
 * linear        z = x weight^T + bias;  output = act(z) + residual
 *               x [rows, in], weight [out, in], bias [out] or NULL,
 *               residual [rows, out] or NULL, output [rows, out]
 * activation    0 none, 1 relu, 2 gelu (z * Phi(z), by the error function)
 * relu_mask     [ceil(out / 64), rows, 8] bytes: bit i of byte j of block c is set
 *               where the derivative of relu at z[64 c + 8 j + i] is one (z > 0, or
 *               NaN); bits past out are not read
 * pre_activation [rows, out] what is kept of z for gelu, an element of the tensors' size
 *               each: the derivative there, a float32 number or a 16-bit code (the
 *               library's own, within 2^-16, small ones within a relative 2^-11)
 * codes, scales an 8-bit checkpoint of x: [rows, pad32(in)] int8 and
 *               [rows, pad32(in) / 32] bytes. 32 values share 2^e, the smallest
 *               power of two with 127 * 2^e at or over their largest magnitude;
 *               the byte is e + 127, or 255 where one of them is an infinity or
 *               NaN: such a block reads back as NaN. code * 2^e is a number of
 *               the tensors' type, so products read back exactly what is kept.
 *               codes start on an 8-byte boundary.
 *
 * Conventions: launches are ordered on `stream`, on the current device; nothing
 * synchronises or allocates. Return 0 or a MUSPACE_E* code with
 * muspace_last_error() set (muspace_msda.h). rows may be 0 (gradients of weight
 * and bias are then zero). in, out at most 2^20; rows below 2^31 - 256; any
 * two of them over at most 2^24 tiles of 128 x 128 (MUSPACE_ERANGE otherwise).
 */
#ifndef MUSPACE_LAYER_H_
#define MUSPACE_LAYER_H_

#include <stddef.h>
#include <stdint.h>

#include "muspace_msda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* relu_mask and pre_activation may be NULL (no gradient wanted); relu_mask is
 * written for activation 1 only, pre_activation for activation 2 only. codes and
 * scales may both be NULL (no checkpoint); an empty output writes none. */
MUSPACE_API int linear_forward(const void *x, int dtype, const void *weight, const void *bias,
                               const void *residual, void *output, uint8_t *relu_mask,
                               void *pre_activation, int8_t *codes, uint8_t *scales, int64_t rows,
                               int64_t in_features, int64_t out_features, int activation,
                               void *stream);

/* The checkpoint alone, the same codes as linear_forward's. */
MUSPACE_API int linear_checkpoint(const void *x, int dtype, int8_t *codes, uint8_t *scales,
                                  int64_t rows, int64_t in_features, void *stream);

/* Bytes of workspace of linear_backward (256-byte aligned; 0: none needed): enough for
 * any set of gradients; _for: for those whose flag is not 0. */
MUSPACE_API size_t linear_backward_workspace_size(int dtype, int64_t rows, int64_t in_features,
                                                  int64_t out_features, int activation);
MUSPACE_API size_t linear_backward_workspace_size_for(int dtype, int64_t rows, int64_t in_features,
                                                      int64_t out_features, int activation,
                                                      int want_input, int want_weight,
                                                      int want_bias);

/* dz = grad_output * act'(z); grad_input = dz weight; grad_weight = dz^T x;
 * grad_bias = sum of dz over rows. A NULL gradient is not computed. x is needed
 * for grad_weight unless codes and scales are given in its place; weight for
 * grad_input; relu_mask for activation 1; pre_activation for activation 2.
 * The gradient of the residual is grad_output itself. Outputs are overwritten. */
MUSPACE_API int linear_backward(const void *grad_output, int dtype, const void *x,
                                const int8_t *codes, const uint8_t *scales, const void *weight,
                                const uint8_t *relu_mask, const void *pre_activation,
                                void *grad_input, void *grad_weight, void *grad_bias,
                                int64_t rows, int64_t in_features, int64_t out_features,
                                int activation, void *workspace, size_t workspace_bytes,
                                void *stream);

/* The gated layer: weight [2 hidden, in] holds the gate's rows, then the others' (bias
 * [2 hidden] or NULL the same); with a and u the two halves of x weight^T + bias,
 *   output = act(a) u   [rows, hidden]
 * activation: 0 none, 1 relu, 2 gelu, 3 silu (a / (1 + exp(-a))), 4 sigmoid. */
MUSPACE_API int gated_linear_forward(const void *x, int dtype, const void *weight,
                                     const void *bias, void *output, int64_t rows,
                                     int64_t in_features, int64_t hidden_features, int activation,
                                     void *stream);

/* Bytes of workspace of gated_linear_backward (256-byte aligned) for the gradients whose
 * flag is not 0. */
MUSPACE_API size_t gated_linear_backward_workspace_size(int dtype, int64_t rows,
                                                        int64_t in_features,
                                                        int64_t hidden_features, int want_input,
                                                        int want_weight, int want_bias);

/* Rows of float32 sums of da and du, [2 hidden] each, that the backward leaves in its workspace
 * for grad_bias (0 for invalid sizes): `aligned` is not 0 where x and weight start on 16-byte
 * boundaries. The workspace's size covers either. */
MUSPACE_API int64_t gated_linear_backward_sum_rows(int dtype, int64_t rows, int64_t in_features,
                                                   int64_t hidden_features, int aligned);

/* a and u are computed again; da = grad_output u act'(a) and du = grad_output act(a) are
 * rounded to the tensors' type (past its range: to infinities); grad_input = [da du]
 * weight, grad_weight = [da du]^T x, grad_bias their sums over the rows. A NULL gradient
 * is not computed; x, weight and bias are needed for any. Outputs are overwritten. */
MUSPACE_API int gated_linear_backward(const void *grad_output, int dtype, const void *x,
                                      const void *weight, const void *bias, void *grad_input,
                                      void *grad_weight, void *grad_bias, int64_t rows,
                                      int64_t in_features, int64_t hidden_features,
                                      int activation, void *workspace, size_t workspace_bytes,
                                      void *stream);

/* Rows in 8 bits: scales[r] = max(max |x[r]| / 127, 2^-126) in float32 (the quotient rounded
 * once), codes[r][c] = x[r][c] / scales[r] rounded to the nearest integer, ties to even (of
 * the float32 quotient), -127 to 127. A row with an infinity or NaN has scale NaN and codes 1.
 * codes [rows, cols], scales [rows]; cols at most 2^20. */
MUSPACE_API int quantize_int8(const void *x, int dtype, int8_t *codes, float *scales, int64_t rows,
                              int64_t cols, void *stream);

/* linear on 8-bit integers: x's rows are quantised as by quantize_int8, weight [out, in]
 * are codes with a scale per row, weight_scales [out] float32:
 *   z = sum of codes * scales[r] * weight_scales[o] + bias;  output = act(z) + residual
 * with sums exact in int32 and the rest in float32, rounded once; activation 0 none,
 * 1 relu, 2 gelu. in at most 2^17. The workspace (256-byte aligned; 0: none needed) holds
 * x's codes and scales. */
MUSPACE_API size_t linear_int8_workspace_size(int dtype, int64_t rows, int64_t in_features,
                                              int64_t out_features);
MUSPACE_API int linear_int8_forward(const void *x, int dtype, const int8_t *weight,
                                    const float *weight_scales, const void *bias,
                                    const void *residual, void *output, int64_t rows,
                                    int64_t in_features, int64_t out_features, int activation,
                                    void *workspace, size_t workspace_bytes, void *stream);

/* layer norm over the last dimension:
 *   c = x - mean(x);  s = 1 / sqrt(mean(c^2) + eps);  output = c s weight + bias
 * x, output [rows, cols]; weight, bias [cols] of weight_dtype (dtype or float32),
 * each may be NULL (ones, zeros). statistics [rows, 2] float32 or NULL: the mean
 * as an offset from the row's first value, and s; or, where the mean is nearer to
 * zero, the mean itself and -s. The backward reads them. */
MUSPACE_API int layer_norm_forward(const void *x, int dtype, const void *weight, const void *bias,
                                   int weight_dtype, void *output, float *statistics, int64_t rows,
                                   int64_t cols, float eps, void *stream);

MUSPACE_API size_t layer_norm_backward_workspace_size(int dtype, int64_t rows, int64_t cols);

/* With h = c s and w = grad_output weight:
 *   grad_input = s (w - mean(w) - h mean(w h));  grad_weight = sum of grad_output h over rows;
 *   grad_bias = sum of grad_output over rows (both of weight_dtype).
 * A NULL gradient is not computed; the workspace is needed for the last two. */
MUSPACE_API int layer_norm_backward(const void *grad_output, int dtype, const void *x,
                                    const void *weight, int weight_dtype, const float *statistics,
                                    void *grad_input, void *grad_weight, void *grad_bias,
                                    int64_t rows, int64_t cols, void *workspace,
                                    size_t workspace_bytes, void *stream);

/* dropout: output = kept ? x / (1 - p) : 0, plus residual (or NULL), over `count`
 * elements. Element i is kept if word i % 4 of Philox4x32-10 at counter (i / 4, offset)
 * (64 bits each, low words first) under the key `seed` is at or over p 2^32, to the
 * nearest. device_seed, where not NULL, is read by the kernel in place of seed: a
 * captured call whose seed changes draws another mask. The gradient of x is the same
 * call on output's gradient, without residual; the residual's is output's own. */
MUSPACE_API int dropout_forward(const void *x, int dtype, const void *residual, void *output,
                                int64_t count, double p, uint64_t seed,
                                const int64_t *device_seed, uint64_t offset, void *stream);

/* The sum of a block with the residual stream, and the norm after it:
 *   y = post_norm(block) (post_norm -1 none: the block; 0 layer, 1 rms)
 *   stream_values = residual_scale residual + gate dropout(y)
 *   output = norm(the same sum, before it is rounded)   (norm 0 layer, 1 rms)
 * block, residual, output, stream_values [rows, cols]; weight, bias, gate, post_weight,
 * post_bias [cols] of weight_dtype (dtype or float32), each may be NULL (ones; biases
 * zeros). The rms norm is x / sqrt(mean(x^2) + eps) weight + bias. dropout is that of
 * dropout_forward over the tensor's elements, p 0 for none. stream_values, statistics
 * and post_statistics ([rows, 4] float32, 16-byte aligned, for the backward) may be
 * NULL. */
MUSPACE_API int residual_norm_forward(const void *block, int dtype, const void *residual,
                                      const void *weight, const void *bias, const void *gate,
                                      const void *post_weight, const void *post_bias,
                                      int weight_dtype, void *output, void *stream_values,
                                      float *statistics, float *post_statistics, int64_t rows,
                                      int64_t cols, int norm, int post_norm, float eps,
                                      float residual_scale, double p, uint64_t seed,
                                      const int64_t *device_seed, uint64_t offset, void *stream);

/* Bytes of workspace of residual_norm_backward (16-byte aligned) for `sums` of the five
 * gradients of weights. */
MUSPACE_API size_t residual_norm_backward_workspace_size(int dtype, int64_t rows, int64_t cols,
                                                         int sums);

/* The gradients from those of output and stream_values (NULL: zeros). A NULL gradient
 * is not computed. 16-bit types read block and residual (stream_values may be NULL);
 * float32 reads stream_values, and block where there is a post norm or grad_gate is
 * wanted (residual, and block otherwise, may be NULL). p, seed, device_seed's value and
 * offset are the forward's. */
MUSPACE_API int residual_norm_backward(
    const void *grad_output, const void *grad_stream, int dtype, const void *block,
    const void *residual, const void *stream_values, const void *weight, const void *gate, const void *post_weight,
    const void *post_bias, int weight_dtype, const float *statistics, const float *post_statistics,
    void *grad_block, void *grad_residual, void *grad_weight, void *grad_bias, void *grad_gate,
    void *grad_post_weight, void *grad_post_bias, int64_t rows, int64_t cols, int norm,
    int post_norm, float residual_scale, double p, uint64_t seed, const int64_t *device_seed,
    uint64_t offset, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MUSPACE_LAYER_H_ */

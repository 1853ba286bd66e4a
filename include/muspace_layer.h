/*
 * C-ABI of the dense operators around deformable attention in an encoder or
 * decoder layer: the linear layer with its epilogue and gradients, its 8-bit
 * input checkpoint, and layer norm with its gradients. Part of
 * `libmuspace_msda.so`, MI355X (gfx950).
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

#ifdef __cplusplus
}
#endif

#endif /* MUSPACE_LAYER_H_ */

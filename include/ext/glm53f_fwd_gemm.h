/* BF16 matrix product with bias, activation and residual in its epilogue, for MI355X (gfx950): the projections of a
 * layer with what follows them, from one row (a decode step) to thousands (a prompt's segment), without a second pass
 * over the outputs. Beside the GEMV and the GEMM for 9 to 64 rows of glm53f_fwd_gemv.h, which give the bare product.
 * The reference has no counterpart (its layers call the GEMM and an elementwise kernel).
 *
 * Conventions (as glm53f_fwd_gemv.h): device pointers; strides in ELEMENTS; the return value is a hipError_t as int32:
 * 0 on success, 1 (hipErrorInvalidValue) when the host rejects an argument, otherwise the launch error. Asynchronous
 * on `stream`, on the current device; nothing is allocated, freed or synchronized inside; may be captured into a graph.
 */
#ifndef GLM53F_FWD_GEMM_H
#define GLM53F_FWD_GEMM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

struct ihipStream_t;

/* The activations of glm53f_fwd_gemm_bf16_fused. */
#define GLM53F_ACT_NONE 0
#define GLM53F_ACT_RELU 1
#define GLM53F_ACT_SILU 2       /* y * sigmoid(y) */
#define GLM53F_ACT_GELU 3       /* y * Phi(y), with the error function */
#define GLM53F_ACT_GELU_TANH 4  /* 0.5 y (1 + tanh(sqrt(2/pi) (y + 0.044715 y^3))) */
#define GLM53F_ACT_SIGMOID 5

/** out[g][m][o] = residual[g][m][o] + act(sum_k x[g][m][k] * w[g][o][k] + bias[g][o])
 *  for g < groups, m < rows, o < n: x row m at x + g*x_gstride + m*ldx, w row o at w + g*w_gstride + o*ldw, bias at
 *  bias + g*b_gstride (bf16, NULL: none), residual at residual + g*r_gstride + m*ldr (of the outputs' type, NULL: none),
 *  out at out + g*o_gstride + m*ldo (bf16, or f32 when out_f32 != 0).
 *  Any rows, n, k from 1 to 2^30 (rows == 0 succeeds without a launch), groups from 1 to 65,535, ldx, ldw >= k, ldo,
 *  ldr >= n, group strides >= 0; pointers aligned to their elements. 16-byte aligned x and w with strides and k that are
 *  multiples of 8 are read fastest, of 128 best.
 *  residual may be out itself with the same strides (the residual stream updated in place); otherwise out overlaps no
 *  input. Outputs of different groups must not overlap.
 *  Numerics: exact bf16 products, f32 sums over k, the epilogue in f32 (an activation of y within 2^-20 (1 + |y|)), one
 *  rounding to the outputs' type. */
int32_t glm53f_fwd_gemm_bf16_fused(const uint16_t* x, int64_t ldx, int64_t x_gstride, const uint16_t* w, int64_t ldw,
                                   int64_t w_gstride, int32_t groups, int32_t rows, int32_t n, int32_t k,
                                   const uint16_t* bias, int64_t b_gstride, int32_t act, const void* residual,
                                   int64_t ldr, int64_t r_gstride, void* out, int32_t out_f32, int64_t ldo,
                                   int64_t o_gstride, struct ihipStream_t* stream);

#ifdef __cplusplus
}
#endif

#endif

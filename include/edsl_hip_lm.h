/*
 * edsl_hip_lm.h -- device-resident operators of language models around the
 * dense layer: the root-mean-square norm, the dense layer on 4-bit weights, and
 * log probabilities of given tokens.
 *
 * No counterpart in the reference, whose programs are dense layers. Calling
 * convention, streams, errors, workspaces and graph capture are those of
 * include/edsl_hip_device.h: device pointers, row strides (ld*) in elements
 * with unit inner stride, work enqueued on `stream`, 0 or an error code with
 * the message in edsl_hip_last_error(). Rows of any length, stride (at least
 * the row) and alignment to their element are taken; a pointer of an optional
 * operand may be null. Sizes go up to 2^30 in each dimension, offsets are 64
 * bits; work beyond one launch (2^31 workgroups) is refused. Sums, maxima and
 * norms are 32-bit floats: rows whose squares, or products with weights, leave
 * their range have results of 0, infinities or NaN. An output may not overlap an input except where
 * stated.
 */
#ifndef EDSL_HIP_LM_H
#define EDSL_HIP_LM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define EDSL_LM_F32 0
#define EDSL_LM_BF16 1
#define EDSL_LM_F16 2
#define EDSL_LM_I8 3   /* integers -127 .. 127 */
#define EDSL_LM_E4M3 4 /* 8-bit floats of 4 exponent and 3 mantissa bits, no infinities */

/* h = x (+ residual);  total = h;  rstd = (mean_n h^2 + eps)^(-1/2);
 * y = h * rstd * weight, for each of M rows of N.
 *
 * x, residual (optional) and total (optional) have type `type` (F32, BF16,
 * F16), weight that type or F32. The norm is that of h in 32 bits, not of the
 * rounded total. y has type `type`, or an 8-bit type with scales[M], one a row:
 * y = q * scales with scales = max_n |y| / Q, Q = 127 (I8) or 448 (E4M3), and
 * q = h * weight * Q / max_n |h * weight| rounded to nearest even (from 32-bit
 * products and a 32-bit quotient); a row of zeros has scale 0, and one whose
 * scale is under 2^-126 codes of 0. A row whose norm is not finite
 * or whose values are NaN has a NaN scale and unspecified codes. rstd[M] is
 * optional, for the backward pass. total may be x or residual, and y may be
 * x, residual or total's memory in the same type and stride. */
int edsl_hip_rms_norm_launch(const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight,
                             int weight_type, void *total, int64_t ldt, void *y, int64_t ldy, int y_type,
                             float *scales, float *rstd, int64_t M, int64_t N, int type, float eps, void *stream);

/* The gradients of the above: h is the total that was normalised, dy the
 * gradient of y, dh (optional) that of total.
 *   t = dy * weight;  dx = rstd * (t - h * rstd * mean_n(t * h * rstd)) + dh
 * is the gradient of x and of residual alike, and dweight[N] (optional, f32)
 * the sum over the rows of dy * h * rstd. Rows are summed in 32 bits in a
 * fixed order: the same call gives the same bits. dy, h, dh and dx have type
 * `type`; dx may be dy, h or dh in the same stride. M = 0 makes dweight 0. */
int edsl_hip_rms_norm_backward_launch(const void *dy, int64_t lddy, const void *h, int64_t ldh, const void *weight,
                                      int weight_type, const float *rstd, const void *dh, int64_t lddh, void *dx,
                                      int64_t lddx, float *dweight, int64_t M, int64_t N, int type, void *stream);

/* Log probabilities of given tokens under softmax(scale * logits) in each of
 * M rows of V logits (F32, BF16, F16), 0 < scale <= 2^127:
 *   lse = log sum_j exp(scale x_j);  logprobs = scale x_token - lse;
 *   entropy = lse - sum_j p_j scale x_j;
 *   top_logprobs, top_ids [M][k]: the k largest, in falling order, equal
 *   logits in the order of their index; k <= EDSL_LM_MAX_TOP and k <= V.
 * tokens and top_ids are int64_t when ids64, else int32_t. A token outside
 * 0 .. V-1 (padding) has log probability 0. logprobs (with tokens), lse,
 * entropy and the top lists (both) are each optional.
 * Logits may be -inf (masked): they have probability 0. A row of nothing else has
 * lse and log probabilities -inf and entropy 0. A row that holds a NaN or +inf
 * has NaN results (but padding's 0) and top_ids -1. V <= 2^21. */
#define EDSL_LM_MAX_TOP 32
int edsl_hip_token_logprobs_launch(const void *logits, int64_t ldl, int type, const void *tokens, int ids64,
                                   float *logprobs, float *lse, float *entropy, float *top_logprobs, void *top_ids,
                                   int k, int64_t M, int64_t V, float scale, void *stream);

/* The gradient of the logits, given those of logprobs (optional, with tokens)
 * and of entropy (optional, with the entropy that the forward pass gave):
 *   dlogits_j = scale * (dlogprobs * ([j == token] - p_j)
 *                        - dentropy * p_j * (scale x_j - lse + entropy)),
 * of the logits' type. A padding token's dlogprobs counts as 0, and so does
 * everything in a row whose lse is -inf. dlogits may be the logits' memory. */
int edsl_hip_token_logprobs_backward_launch(const void *logits, int64_t ldl, int type, const void *tokens, int ids64,
                                            const float *lse, const float *dlogprobs, const float *entropy,
                                            const float *dentropy, void *dlogits, int64_t lddl, int64_t M, int64_t V,
                                            float scale, void *stream);

/* The dense layer on 4-bit weights with a scale and, optionally, a zero point
 * for each column and group of `group` successive k (32, 64 or a multiple of
 * 128; the last group may be shorter):
 *   W[k][n] = scales[k / group][n] * (q[k][n] - zeros[k / group][n]),
 * q and zeros integers 0 .. 15 (the low four bits of their bytes), zeros 8 where
 * there are none. K <= 2^23. edsl_hip_q4_pack_launch lays the weights out once, in
 * edsl_hip_q4_packed_bytes bytes (-1: arguments that it does not take, with the
 * message in edsl_hip_last_error) at a 256-byte aligned address; scales are F32,
 * BF16 or F16 and kept as they are. */
int64_t edsl_hip_q4_packed_bytes(int64_t K, int64_t N, int group, int scale_type, int has_zeros);
int edsl_hip_q4_pack_launch(const uint8_t *q, int64_t ldq, const void *scales, int64_t lds, int scale_type,
                            const uint8_t *zeros, int64_t ldz, int64_t K, int64_t N, int group, void *packed,
                            size_t packed_bytes, void *stream);

/* Y[M,N] = epilogue(x_scales[m] * X[M,K] @ W (+ bias)), EDSL_EPI_* epilogues of
 * include/edsl_hip_device.h. X is F32, BF16, F16, I8 or E4M3, x_scales[M] (f32)
 * optional; Y is F32, BF16 or F16, bias[N] of any of these; K, N, group,
 * scale_type and has_zeros as packed. Products are exact and sums 32-bit: no
 * weight or activation is rounded, f32 ones included. X of 16 and 8 bits meets
 * weights held as 16 + q, less its sum times 16 + zero, so that the sums' roundings
 * are those of terms of |x| scale (32 + q + zero). Sums are taken in a fixed
 * order. A row of X that holds an infinity or NaN gives NaN in all of Y's row, but
 * 0 with the epilogues that select (IF_RELU, y > 0 ? y : 0): NaN is not above 0. */
int edsl_hip_q4_dense_launch(const void *X, int64_t ldx, int x_type, const float *x_scales, const void *packed,
                             const void *bias, int bias_type, void *Y, int64_t ldy, int y_type, int64_t M, int64_t N,
                             int64_t K, int group, int scale_type, int has_zeros, int epilogue, float alpha,
                             void *stream);

#ifdef __cplusplus
}
#endif

#endif /* EDSL_HIP_LM_H */

/*
 * edsl_hip_lm.h -- device-resident operators of language models around the
 * dense layer: the root-mean-square norm, the dense layer on 4-bit weights, in
 * 8-bit integers and on groups of rows, log probabilities of given tokens, and
 * sampling.
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

/* The dense layer in 8-bit integers, a scale for each column of W and, optionally,
 * each row of X:
 *   Y[m][n] = epilogue(x_scales[m] * scales[n] * sum_k X[m][k] q[k][n] (+ bias[n])).
 * Sums are 32-bit integers and exact: 1 <= K < 2^17, values -128 .. 127. The sum is rounded to
 * f32 once and then multiplied by scales[n] and by x_scales[m]. edsl_hip_i8_pack_launch
 * lays q[K][N] and scales[N] (F32, BF16, F16) out once, in
 * edsl_hip_i8_packed_bytes bytes (-1: arguments that it does not take) at a 256-byte
 * aligned address. Y is F32, BF16 or F16, bias of any of these. */
int64_t edsl_hip_i8_packed_bytes(int64_t K, int64_t N);
int edsl_hip_i8_pack_launch(const int8_t *q, int64_t ldq, const void *scales, int scale_type, int64_t K, int64_t N,
                            void *packed, size_t packed_bytes, void *stream);
int edsl_hip_i8_dense_launch(const int8_t *X, int64_t ldx, const float *x_scales, const void *packed, const void *bias,
                             int bias_type, void *Y, int64_t ldy, int y_type, int64_t M, int64_t N, int64_t K,
                             int epilogue, float alpha, void *stream);

/* The dense layer on groups of rows, each with weights of its own (experts):
 *   Y[r] = epilogue(X[r] @ W[e] (+ bias[e]))   for offsets[e] <= r < offsets[e+1].
 * X is [T][K], W [E][K][N] (w_stride elements from one group to the next; where
 * w_turned, each is held as [N][K] with rows of ldw), bias [E][N] with rows of ldbias
 * (0: one for all), Y [T][N], all of `type` (F32, BF16, F16). offsets[E+1] is
 * device memory, int64_t when ids64, else int32_t; it rises from 0 or more to T or less, and may
 * leave groups empty. Rows before the first and behind the last group are left as they are.
 * Offsets outside 0 .. T are cut to it and falling ones make empty groups: nothing
 * outside the operands is read or written, but which rows are is then unspecified.
 * E <= 65535. Y may not overlap an input. Sums are 32-bit floats in a fixed order, rounded once to `type`
 * after the epilogue. */
int edsl_hip_grouped_dense_launch(const void *X, int64_t ldx, const void *W, int64_t ldw, int64_t w_stride,
                                  int w_turned, const void *offsets, int ids64, int64_t E, const void *bias,
                                  int64_t ldbias, void *Y, int64_t ldy, int64_t T, int64_t N, int64_t K, int type,
                                  int epilogue, float alpha, void *stream);

/* Its gradients, each optional. With dZ = dY where there is no activation, else
 * dY * (Y > 0 ? 1 : slope), slope 0 or the leaky epilogue's alpha (>= 0; where it is 0, dZ is 0 whatever dY holds),
 * rounded to `type` for dX and, where that is BF16 or F32, for dW of that type (Y is what the forward pass gave, and may be
 * null without an activation):
 *   dX[r] = dZ[r] @ W[e]^T;  dW[e] = sum over the group's rows of X[r]^T dZ[r];
 *   db[e] = sum of dZ[r], without that rounding.
 * dX has `type`, dW and db that or F32 (dw_type, db_type); dW is [E][K][N], or turned as W
 * may be. Groups without rows have dW and db 0; rows of no group leave dX as it is.
 * dW in F32 or F16 through a slope of 16-bit dY is the sum of two products, of dY where Y > 0 and of dY elsewhere, that
 * one times the slope. An output may not overlap an input or another output. The same call gives the same bits. */
int edsl_hip_grouped_dense_backward_launch(const void *dY, int64_t lddy, const void *X, int64_t ldx, const void *W,
                                           int64_t ldw, int64_t w_stride, int w_turned, const void *offsets, int ids64,
                                           int64_t E, const void *Y, int64_t ldy, void *dX, int64_t lddx, void *dW,
                                           int64_t lddw, int64_t dw_stride, int dw_turned, int dw_type, void *db,
                                           int64_t lddb, int db_type, int64_t T, int64_t N, int64_t K, int type,
                                           int epilogue, float alpha, void *stream);

/* Draws a token for each of M rows of V logits (F32, BF16, F16) with given numbers
 * uniforms[M] in [0, 1). With w_i = exp((x_i - max x) / temperature), kept are
 *   the top_k largest logits, equal ones in the order of their index;
 *   of these, in falling order, those with less than top_p of their mass before them;
 *   of these, the ones with w_i >= min_p;
 * and the token is the first index at which the running sum of the kept w_i, by index,
 * exceeds uniforms[m] times the whole of it. Temperature 0 takes the largest logit, the first of
 * equal ones. top_k <= 0 or >= V, top_p >= 1 and min_p <= 0 leave their step out; the largest
 * logit is always kept. logprobs[M] (optional) is the log probability with which the token was drawn.
 * Each setting is one for all rows (`_all`) or, where its pointer is not null, M of them.
 * w_i are held in units of 2^-46 (2^(ceil(log2 V) - 62) for V beyond 2^16), to nearest, and sums
 * are exact: the same call gives the same tokens. Logits of -inf are never drawn; a row of
 * nothing else gives token -1 and log probability -inf, and one that holds NaN or +inf, or whose
 * settings or number are NaN or whose temperature is negative or infinite, -1 and NaN. Numbers outside [0, 1) count as
 * the nearest inside. tokens are int64_t when ids64, else int32_t. V <= 2^21. */
int edsl_hip_sample_tokens_launch(const void *logits, int64_t ldl, int type, const float *uniforms, void *tokens,
                                  int ids64, float *logprobs, const float *temperature, float temperature_all,
                                  const int32_t *top_k, int top_k_all, const float *top_p, float top_p_all,
                                  const float *min_p, float min_p_all, int64_t M, int64_t V, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* EDSL_HIP_LM_H */

/*
 * bbh_int8.h - the engine's 8-bit operators: rows quantised with one scale
 * each, norms that write 8-bit rows, and the Linear on 8-bit integers.
 *
 * No counterpart in the reference, which is fp16 throughout.  They stand next
 * to bbh_linear and bbh_layernorm for callers that serve a model, or keep an
 * index of embeddings, in 8 bits.  All conventions of bbh.h hold (device
 * pointers, row-major contiguous operands, `stream`, bbh_status,
 * bbh_last_error; nothing allocates, so every call can be captured into a
 * HIP graph).
 *
 * An 8-bit row is D int8 codes in [-127, 127] and one fp32 scale; it stands
 * for code * scale.  Quantising is symmetric: with a = max_j |x_j|,
 *   scale = a / 127,  code_j = x_j / scale rounded to nearest, ties to even.
 * A row of zeros has scale 0 and codes 0.  A row that holds an infinity or a
 * NaN has scale NaN and codes 0, so that whatever reads it is NaN too.
 */
#ifndef BBH_INT8_H
#define BBH_INT8_H

#include "bbh.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Longest row: 128 * 128 * 131071 < 2^31, so no sum of products of int8 codes
 * (-128 included) leaves int32. */
#define BBH_I8_MAX_K 131071
/* Longest row of the norms below (a row stays in one workgroup's registers). */
#define BBH_I8_MAX_NORM 16384

/* q (M, D) int8 and scale (M) fp32 of x (M, D) fp16; D <= BBH_I8_MAX_K.  The
 * codes are the exact quotients 127 x / a rounded once.  For activations (a
 * scale a token), weights (N, K) (a scale an output channel) and embeddings. */
bbh_status bbh_quantize_rows(const void *x, int8_t *q, float *scale, int M, int D,
                             bbh_stream_t stream);
/* x (M, D) fp16 = q * scale in fp32, rounded to fp16; D <= BBH_I8_MAX_K.  Any int8
 * codes. */
bbh_status bbh_dequantize_rows(const int8_t *q, const float *scale, void *x, int M, int D,
                               bbh_stream_t stream);

/* Norms with the residual's addition and an 8-bit output, D <= BBH_I8_MAX_NORM,
 * eps >= 0.  With h = x + residual (residual may be NULL) kept in fp32:
 *   bbh_rmsnorm_quantize    v = h / sqrt(mean(h^2) + eps) * gamma
 *   bbh_layernorm_quantize  v = (h - mean(h)) / sqrt(var(h) + eps) * gamma + beta
 * q and scale are the quantised rows of v as it is in fp32 (not of the fp16 y).
 * sum (optional, fp16) gets h, the residual stream of a pre-norm block; y
 * (optional, fp16) gets v, which a post-norm block adds later.  x, residual,
 * gamma, beta: fp16.  sum and y may each be x or residual, but not each other;
 * q and scale overlap nothing.  With eps 0 a row of zeros (rmsnorm) or of equal
 * values (layernorm) is the formula's 0 / 0: a row with a NaN.  Sums are fp32, in
 * an order that goes with D and M, so a row's last bits may differ with the number
 * of rows it is among (its codes where a value lies at a tie). */
bbh_status bbh_rmsnorm_quantize(const void *x, const void *residual, const void *gamma,
                                void *sum, void *y, int8_t *q, float *scale, int M, int D,
                                float eps, bbh_stream_t stream);
bbh_status bbh_layernorm_quantize(const void *x, const void *residual, const void *gamma,
                                  const void *beta, void *sum, void *y, int8_t *q,
                                  float *scale, int M, int D, float eps, bbh_stream_t stream);

/* bbh_linear on 8-bit rows: C(M,N) fp16 = a_scale[m] * b_scale[n] *
 * sum_k A[m,k] B[n,k] [+ bias[n]] [then GELU]; A (M, K) and B (N, K) int8,
 * a_scale (M) and b_scale (N) fp32, bias (N) fp16 or NULL.  The sum is exact in
 * int32, the rest fp32 (the sum times a_scale, that times b_scale), rounded to fp16
 * once, so a result does not depend on M or on how the work is split.  GELU is
 * within 7.6e-5 of the exact-erf form for values of any size; that is absolute: of
 * values below about -4.1, whose GELU is as small, no digit need be right (-3.0e-5
 * from -4.5 on).  Any M, N >= 1 and 1 <= K <= BBH_I8_MAX_K, any alignment
 * of A and B (of which, where it is no multiple of 4, the 4-byte words around
 * the first and last bytes are read); fastest where K and the addresses of A and
 * B are multiples of 16, then of 4. */
bbh_status bbh_linear_i8(const int8_t *A, const float *a_scale, const int8_t *B,
                         const float *b_scale, void *C, int M, int N, int K, const void *bias,
                         int gelu, bbh_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* BBH_INT8_H */

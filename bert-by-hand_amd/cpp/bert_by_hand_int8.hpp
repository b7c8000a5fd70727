// bert_by_hand_int8.hpp - the 8-bit operators (include/bbh_int8.h) in the C++
// layer's manner: default arguments, an optional trailing stream, and errors
// that print and abort.  No counterpart in the reference.
#pragma once

#include "bert_by_hand.hpp"
#include "bbh_int8.h"

// q (M, D), scale (M) = 8-bit rows of x (M, D): scale = max |row| / 127.
inline void launch_quantize_rows(const __half *x, int8_t *q, float *scale, int M, int D,
                                 hipStream_t stream = nullptr) {
  BBH_CHECK(bbh_quantize_rows(x, q, scale, M, D, stream));
}

// x (M, D) = q * scale.
inline void launch_dequantize_rows(const int8_t *q, const float *scale, __half *x, int M, int D,
                                   hipStream_t stream = nullptr) {
  BBH_CHECK(bbh_dequantize_rows(q, scale, x, M, D, stream));
}

// 8-bit rows of the RMS norm of x (+ residual); sum (x + residual) and y (the
// norm) are written where given.
inline void launch_rmsnorm_quantize(const __half *x, const __half *gamma, int8_t *q, float *scale,
                                    int M, int D, float eps, const __half *residual = nullptr,
                                    __half *sum = nullptr, __half *y = nullptr,
                                    hipStream_t stream = nullptr) {
  BBH_CHECK(bbh_rmsnorm_quantize(x, residual, gamma, sum, y, q, scale, M, D, eps, stream));
}

// The same of the LayerNorm.
inline void launch_layernorm_quantize(const __half *x, const __half *gamma, const __half *beta,
                                      int8_t *q, float *scale, int M, int D, float eps,
                                      const __half *residual = nullptr, __half *sum = nullptr,
                                      __half *y = nullptr, hipStream_t stream = nullptr) {
  BBH_CHECK(
      bbh_layernorm_quantize(x, residual, gamma, beta, sum, y, q, scale, M, D, eps, stream));
}

// launch_matmul on 8-bit rows: C = a_scale b_scale (A . B^T) (+ bias) (then GELU).
inline void launch_matmul_i8(const int8_t *A, const float *a_scale, const int8_t *B,
                             const float *b_scale, __half *C, int M, int N, int K,
                             const __half *bias = nullptr, bool gelu = false,
                             hipStream_t stream = nullptr) {
  BBH_CHECK(bbh_linear_i8(A, a_scale, B, b_scale, C, M, N, K, bias, gelu ? 1 : 0, stream));
}

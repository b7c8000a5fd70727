// Host launchers of the 8-bit operators (quantize.hip, gemm_i8.hip).  As in
// kernels.h each enqueues on `s` and returns the launch status; the argument
// checks are in capi_int8.hip.
#pragma once

#include "common.h"

namespace bbh {

constexpr int kMaxI8Row = 131071;   // 128 * 128 * K < 2^31
constexpr int kMaxNormRow = 16384;  // a row of the norms stays in registers

// q, scale = 8-bit rows of x (M, D); D <= kMaxI8Row.
hipError_t quantize_rows(const f16* x, int8_t* q, float* scale, int M, int D, hipStream_t s);
hipError_t dequantize_rows(const int8_t* q, const float* scale, f16* x, int M, int D,
                           hipStream_t s);

// h = x [+ residual] in fp32, its RMS norm (beta null) or LayerNorm, and that
// quantised; sum (h) and y (the norm) are written in fp16 where not null.
// D <= kMaxNormRow.
hipError_t rmsnorm_quantize(const f16* x, const f16* residual, const f16* gamma, f16* sum, f16* y,
                            int8_t* q, float* scale, int M, int D, float eps, hipStream_t s);
hipError_t layernorm_quantize(const f16* x, const f16* residual, const f16* gamma,
                              const f16* beta, f16* sum, f16* y, int8_t* q, float* scale, int M,
                              int D, float eps, hipStream_t s);

// C(M,N) = fp16(sa[m] sb[n] sum_k A(M,K) B(N,K) [+ bias] [GELU]), int8 operands.
hipError_t gemm_i8(const int8_t* A, const float* sa, const int8_t* B, const float* sb,
                   const f16* bias, f16* C, int M, int N, int K, bool gelu, hipStream_t s);

}  // namespace bbh

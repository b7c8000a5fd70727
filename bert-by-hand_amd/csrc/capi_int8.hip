// C ABI of the 8-bit operators (include/bbh_int8.h): argument validation.

#include <math.h>

#include <string>

#include "../../include/bbh_int8.h"
#include "int8.h"

using bbh::f16;

namespace bbh_detail {
bbh_status set_error(bbh_status s, const std::string& msg);  // capi.hip
}

static_assert(bbh::kMaxI8Row == BBH_I8_MAX_K && bbh::kMaxNormRow == BBH_I8_MAX_NORM, "limits");

namespace {

bbh_status fail(bbh_status s, const char* what, const char* msg) {
  return bbh_detail::set_error(s, std::string(what) + ": " + msg);
}

bbh_status done(hipError_t e, const char* what) {
  if (e == hipSuccess) return BBH_OK;
  return bbh_detail::set_error(BBH_ERR_HIP, std::string(what) + ": " + hipGetErrorName(e) + " (" +
                                                hipGetErrorString(e) + ")");
}

template <class T>
bool off(const T* p, uintptr_t n) {
  return ((uintptr_t)p & (n - 1)) != 0;
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x < y + nb && y < x + na;
}

bbh_status rows(const char* what, int M, int D, int max) {
  if (M < 1 || D < 1) return fail(BBH_ERR_INVALID_ARG, what, "M and D must be positive");
  if (D > max)
    return bbh_detail::set_error(
        BBH_ERR_UNSUPPORTED,
        std::string(what) + ": rows longer than " + std::to_string(max) + " are not supported");
  return BBH_OK;
}

bbh_status norm_args(const char* what, const void* x, const void* residual, const void* gamma,
                     const void* beta, void* sum, void* y, int8_t* q, float* scale, int M, int D,
                     float eps) {
  if (!x || !gamma || !q || !scale) return fail(BBH_ERR_INVALID_ARG, what, "null argument");
  const bbh_status s = rows(what, M, D, BBH_I8_MAX_NORM);
  if (s != BBH_OK) return s;
  if (!(eps >= 0.f) || !isfinite(eps))
    return fail(BBH_ERR_INVALID_ARG, what, "eps must be finite and not negative");
  for (const void* p : {x, residual, gamma, beta, (const void*)sum, (const void*)y})
    if (off((const char*)p, 2)) return fail(BBH_ERR_INVALID_ARG, what, "fp16 operands must be 2-byte aligned");
  if (off(scale, 4)) return fail(BBH_ERR_INVALID_ARG, what, "scale must be 4-byte aligned");
  const size_t n = (size_t)M * D, halves = 2 * n, col = 2 * (size_t)D;
  // an output that is exactly x or residual is read before it is written
  for (const void* o : {(const void*)sum, (const void*)y})
    for (const void* i : {x, residual})
      if (o != i && overlap(o, halves, i, halves))
        return fail(BBH_ERR_INVALID_ARG, what, "sum or y overlaps x or residual in part");
  if (overlap(sum, halves, y, halves))
    return fail(BBH_ERR_INVALID_ARG, what, "sum and y overlap");
  for (const void* o : {(const void*)sum, (const void*)y})
    if (overlap(o, halves, gamma, col) || overlap(o, halves, beta, col))
      return fail(BBH_ERR_INVALID_ARG, what, "sum or y overlaps gamma or beta");
  for (const void* p : {x, residual, (const void*)sum, (const void*)y})
    if (overlap(q, n, p, halves) || overlap(scale, 4 * (size_t)M, p, halves))
      return fail(BBH_ERR_INVALID_ARG, what, "q or scale overlaps another operand");
  if (overlap(q, n, gamma, col) || overlap(q, n, beta, col) ||
      overlap(scale, 4 * (size_t)M, gamma, col) || overlap(scale, 4 * (size_t)M, beta, col) ||
      overlap(q, n, scale, 4 * (size_t)M))
    return fail(BBH_ERR_INVALID_ARG, what, "q or scale overlaps another operand");
  return BBH_OK;
}

}  // namespace

extern "C" {

bbh_status bbh_quantize_rows(const void* x, int8_t* q, float* scale, int M, int D,
                             bbh_stream_t stream) {
  const char* what = "bbh_quantize_rows";
  if (!x || !q || !scale) return fail(BBH_ERR_INVALID_ARG, what, "null argument");
  const bbh_status s = rows(what, M, D, BBH_I8_MAX_K);
  if (s != BBH_OK) return s;
  if (off((const char*)x, 2) || off(scale, 4))
    return fail(BBH_ERR_INVALID_ARG, what, "x must be 2-byte and scale 4-byte aligned");
  const size_t n = (size_t)M * D;
  if (overlap(q, n, x, 2 * n) || overlap(scale, 4 * (size_t)M, x, 2 * n) ||
      overlap(q, n, scale, 4 * (size_t)M))
    return fail(BBH_ERR_INVALID_ARG, what, "operands overlap");
  return done(bbh::quantize_rows(static_cast<const f16*>(x), q, scale, M, D,
                                 static_cast<hipStream_t>(stream)),
              what);
}

bbh_status bbh_dequantize_rows(const int8_t* q, const float* scale, void* x, int M, int D,
                               bbh_stream_t stream) {
  const char* what = "bbh_dequantize_rows";
  if (!q || !scale || !x) return fail(BBH_ERR_INVALID_ARG, what, "null argument");
  const bbh_status s = rows(what, M, D, BBH_I8_MAX_K);
  if (s != BBH_OK) return s;
  if (off((const char*)x, 2) || off(scale, 4))
    return fail(BBH_ERR_INVALID_ARG, what, "x must be 2-byte and scale 4-byte aligned");
  const size_t n = (size_t)M * D;
  if (overlap(x, 2 * n, q, n) || overlap(x, 2 * n, scale, 4 * (size_t)M))
    return fail(BBH_ERR_INVALID_ARG, what, "operands overlap");
  return done(bbh::dequantize_rows(q, scale, static_cast<f16*>(x), M, D,
                                   static_cast<hipStream_t>(stream)),
              what);
}

bbh_status bbh_rmsnorm_quantize(const void* x, const void* residual, const void* gamma, void* sum,
                                void* y, int8_t* q, float* scale, int M, int D, float eps,
                                bbh_stream_t stream) {
  const char* what = "bbh_rmsnorm_quantize";
  const bbh_status s = norm_args(what, x, residual, gamma, nullptr, sum, y, q, scale, M, D, eps);
  if (s != BBH_OK) return s;
  return done(bbh::rmsnorm_quantize(static_cast<const f16*>(x), static_cast<const f16*>(residual),
                                    static_cast<const f16*>(gamma), static_cast<f16*>(sum),
                                    static_cast<f16*>(y), q, scale, M, D, eps,
                                    static_cast<hipStream_t>(stream)),
              what);
}

bbh_status bbh_layernorm_quantize(const void* x, const void* residual, const void* gamma,
                                  const void* beta, void* sum, void* y, int8_t* q, float* scale,
                                  int M, int D, float eps, bbh_stream_t stream) {
  const char* what = "bbh_layernorm_quantize";
  if (!beta) return fail(BBH_ERR_INVALID_ARG, what, "null argument");
  const bbh_status s = norm_args(what, x, residual, gamma, beta, sum, y, q, scale, M, D, eps);
  if (s != BBH_OK) return s;
  return done(bbh::layernorm_quantize(
                  static_cast<const f16*>(x), static_cast<const f16*>(residual),
                  static_cast<const f16*>(gamma), static_cast<const f16*>(beta),
                  static_cast<f16*>(sum), static_cast<f16*>(y), q, scale, M, D, eps,
                  static_cast<hipStream_t>(stream)),
              what);
}

bbh_status bbh_linear_i8(const int8_t* A, const float* a_scale, const int8_t* B,
                         const float* b_scale, void* C, int M, int N, int K, const void* bias,
                         int gelu, bbh_stream_t stream) {
  const char* what = "bbh_linear_i8";
  if (!A || !a_scale || !B || !b_scale || !C)
    return fail(BBH_ERR_INVALID_ARG, what, "null operand");
  if (M < 1 || N < 1 || K < 1)
    return fail(BBH_ERR_INVALID_ARG, what, "M, N, K must be positive");
  if (K > BBH_I8_MAX_K)
    return fail(BBH_ERR_UNSUPPORTED, what, "K above 131071: sums could leave int32");
  if (off(a_scale, 4) || off(b_scale, 4) || off((const char*)C, 2) || off((const char*)bias, 2))
    return fail(BBH_ERR_INVALID_ARG, what, "scales must be 4-byte, C and bias 2-byte aligned");
  const size_t nc = (size_t)M * N * 2;
  if (overlap(C, nc, A, (size_t)M * K) || overlap(C, nc, B, (size_t)N * K) ||
      overlap(C, nc, a_scale, 4 * (size_t)M) || overlap(C, nc, b_scale, 4 * (size_t)N) ||
      overlap(C, nc, bias, 2 * (size_t)N))
    return fail(BBH_ERR_INVALID_ARG, what, "C overlaps an operand");
  return done(bbh::gemm_i8(A, a_scale, B, b_scale, static_cast<const f16*>(bias),
                           static_cast<f16*>(C), M, N, K, gelu != 0,
                           static_cast<hipStream_t>(stream)),
              what);
}

}  // extern "C"

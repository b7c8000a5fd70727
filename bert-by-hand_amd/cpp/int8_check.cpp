// The 8-bit operators through the C++ layer: a small Linear from fp16 rows and
// weights (quantise both, multiply, read the rows back), and the two norms,
// against the formulas in double on the host.  Prints one line per case and
// exits non-zero when any fails.
#include <cmath>
#include <cstdio>
#include <vector>

#include "bert_by_hand_int8.hpp"

namespace {

int failures = 0;

void report(const char* tag, double worst) {  // worst error over its bound
  const bool pass = worst <= 1.0;
  std::printf("[%s] error / bound = %.3f %s\n", tag, worst, pass ? "PASS" : "FAIL");
  if (!pass) ++failures;
}

// Values of both signs between -2 and 2, no two rows alike.
std::vector<__half> values(size_t n, uint32_t seed) {
  std::vector<__half> v(n);
  for (auto& x : v) {
    seed = seed * 1664525u + 1013904223u;
    x = __float2half((float)(seed >> 8) / (1 << 22) - 2.0f);
  }
  return v;
}

template <class T>
DeviceBuffer upload(const std::vector<T>& v) {
  DeviceBuffer b(v.size() * sizeof(T));
  b.from_host(v.data(), v.size() * sizeof(T));
  return b;
}

template <class T>
std::vector<T> download(const DeviceBuffer& b) {
  std::vector<T> v(b.bytes() / sizeof(T));
  b.to_host(v.data(), b.bytes());
  return v;
}

struct Rows {  // 8-bit rows on the device and the host
  DeviceBuffer q, scale;
  Rows(size_t m, size_t d) : q(m * d), scale(m * sizeof(float)) {}
  int8_t* codes() { return static_cast<int8_t*>(q.data()); }
  float* scales() { return static_cast<float*>(scale.data()); }
};

__half* halves(DeviceBuffer& b) { return static_cast<__half*>(b.data()); }

// Worst error of 8-bit rows against v (m, d), over half a scale and the fp32
// error of the norms (2^-17 of the row's largest value covers it here).
double rows_error(const Rows& r, const std::vector<double>& v, int m, int d) {
  const auto q = download<int8_t>(r.q);
  const auto s = download<float>(r.scale);
  double worst = 0;
  for (int i = 0; i < m; ++i) {
    double a = 0;
    for (int j = 0; j < d; ++j) a = std::fmax(a, std::fabs(v[(size_t)i * d + j]));
    for (int j = 0; j < d; ++j) {
      const double e = std::fabs(q[(size_t)i * d + j] * (double)s[i] - v[(size_t)i * d + j]);
      worst = std::fmax(worst, e / (a / 254 + a / 131072));
    }
  }
  return worst;
}

}  // namespace

int main() {
  const int M = 37, N = 70, K = 301;
  const auto x = values((size_t)M * K, 1), w = values((size_t)N * K, 2), bias = values(N, 3);
  DeviceBuffer dx = upload(x), dw = upload(w), db = upload(bias);
  Rows a(M, K), b(N, K);
  DeviceBuffer back((size_t)M * K * sizeof(__half)), c((size_t)M * N * sizeof(__half));
  launch_quantize_rows(halves(dx), a.codes(), a.scales(), M, K);
  launch_quantize_rows(halves(dw), b.codes(), b.scales(), N, K);
  launch_dequantize_rows(a.codes(), a.scales(), halves(back), M, K);
  launch_matmul_i8(a.codes(), a.scales(), b.codes(), b.scales(), halves(c), M, N, K, halves(db));

  std::vector<double> v(x.size());
  for (size_t i = 0; i < x.size(); ++i) v[i] = __half2float(x[i]);
  report("quantize_rows", rows_error(a, v, M, K));

  const auto qa = download<int8_t>(a.q), qb = download<int8_t>(b.q);
  const auto sa = download<float>(a.scale), sb = download<float>(b.scale);
  const auto hx = download<__half>(back), hc = download<__half>(c);
  double worst = 0;
  for (size_t i = 0; i < hx.size(); ++i) {  // one fp16 rounding of an fp32 product
    const double want = qa[i] * (double)sa[i / K];
    worst = std::fmax(worst, std::fabs(__half2float(hx[i]) - want) /
                                 (std::fabs(want) * (1.0 / 2048 + 1e-7) + 3e-8));
  }
  report("dequantize_rows", worst);
  worst = 0;
  for (int m = 0; m < M; ++m)
    for (int n = 0; n < N; ++n) {
      long acc = 0;
      for (int k = 0; k < K; ++k) acc += (long)qa[(size_t)m * K + k] * qb[(size_t)n * K + k];
      const double p = acc * (double)sa[m] * sb[n], want = p + __half2float(bias[n]);
      // three fp32 roundings, then fp16
      const double bound = std::fabs(p) * 3e-7 + std::fabs(want) * (1.0 / 2048 + 1e-7) + 3e-8;
      worst = std::fmax(worst, std::fabs(__half2float(hc[(size_t)m * N + n]) - want) / bound);
    }
  report("matmul_i8", worst);

  const auto r = values((size_t)M * K, 4), g = values(K, 5), be = values(K, 6);
  DeviceBuffer dr = upload(r), dg = upload(g), dbe = upload(be);
  for (int ln = 0; ln < 2; ++ln) {
    Rows o(M, K);
    if (ln)
      launch_layernorm_quantize(halves(dx), halves(dg), halves(dbe), o.codes(), o.scales(), M, K,
                                1e-5f, halves(dr));
    else
      launch_rmsnorm_quantize(halves(dx), halves(dg), o.codes(), o.scales(), M, K, 1e-5f,
                              halves(dr));
    for (int m = 0; m < M; ++m) {
      const size_t at = (size_t)m * K;
      double mean = 0, var = 0;
      for (int k = 0; k < K; ++k) v[at + k] = (double)__half2float(x[at + k]) + __half2float(r[at + k]);
      for (int k = 0; ln && k < K; ++k) mean += v[at + k] / K;
      for (int k = 0; k < K; ++k) var += (v[at + k] - mean) * (v[at + k] - mean) / K;
      for (int k = 0; k < K; ++k)
        v[at + k] = (v[at + k] - mean) / std::sqrt(var + (double)1e-5f) * __half2float(g[k]) +
                    (ln ? __half2float(be[k]) : 0.0f);
    }
    report(ln ? "layernorm_quantize" : "rmsnorm_quantize", rows_error(o, v, M, K));
  }
  std::printf("%d failure(s)\n", failures);
  return failures != 0;
}

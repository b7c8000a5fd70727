// Rotary positions and attention through the C++ layer: rows of q, k and v normed and rotated into
// q and the slots of a cache, then causal attention of a prompt and of one token more over the
// cache, against the formulas in double on the host.  Prints one line per case and exits non-zero
// when any fails.
#include <cmath>
#include <cstdio>
#include <vector>

#include "bert_by_hand_attend.hpp"

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

__half* halves(DeviceBuffer& b) { return static_cast<__half*>(b.data()); }

constexpr int kHeads = 6, kKv = 2, kDim = 64, kTokens = 45, kSlots = 60;
constexpr int kWidth = (kHeads + 2 * kKv) * kDim;  // a fused row: q, k, v

// Head h (of fused row i) normed by gamma and turned to position i, in double.
std::vector<double> turned(const std::vector<__half>& x, int i, int h, const std::vector<__half>& gamma) {
  std::vector<double> v(kDim);
  double sq = 0;
  for (int d = 0; d < kDim; ++d) {
    v[d] = __half2float(x[(size_t)i * kWidth + h * kDim + d]);
    sq += v[d] * v[d] / kDim;
  }
  for (int d = 0; d < kDim; ++d) v[d] *= __half2float(gamma[d]) / std::sqrt(sq + (double)1e-6f);
  for (int p = 0; p < kDim / 2; ++p) {
    const double t = i * std::pow(10000.0, -2.0 * p / kDim);
    const double a = v[p], b = v[p + kDim / 2];
    v[p] = a * std::cos(t) - b * std::sin(t);
    v[p + kDim / 2] = b * std::cos(t) + a * std::sin(t);
  }
  return v;
}

// Of values up to `size`: one fp16 rounding, and fp32's before it.
double bound(double value, double size) { return std::fabs(value) / 2048 + size * 4e-6 + 1e-7; }

}  // namespace

int main() {
  const auto x = values((size_t)kTokens * kWidth, 1), gq = values(kDim, 2), gk = values(kDim, 3);
  DeviceBuffer dx = upload(x), dgq = upload(gq), dgk = upload(gk);
  DeviceBuffer q((size_t)kTokens * kHeads * kDim * sizeof(__half)), out(q.bytes());
  DeviceBuffer kc((size_t)kSlots * kKv * kDim * sizeof(__half)), vc(kc.bytes());
  std::vector<int64_t> slots(kTokens);
  for (int i = 0; i < kTokens; ++i) slots[i] = i;
  DeviceBuffer dslots = upload(slots);

  Rope first(kDim), rope(std::move(first));
  bbh_rope_args a = rope_args(heads_of(halves(dx), kHeads, kDim, kWidth), kTokens, kHeads, kDim, kTokens);
  a.q_out = heads_of(halves(q), kHeads, kDim);
  a.k = heads_of(halves(dx) + kHeads * kDim, kKv, kDim, kWidth);
  a.v = heads_of(halves(dx) + (kHeads + kKv) * kDim, kKv, kDim, kWidth);
  a.k_out = heads_of(halves(kc), kKv, kDim);
  a.v_out = heads_of(halves(vc), kKv, kDim);
  a.kv_heads = kKv;
  a.q_gamma = dgq.data();
  a.k_gamma = dgk.data();
  a.kv_rows = static_cast<const int64_t*>(dslots.data());
  a.kv_out_rows = kSlots;
  launch_rope(rope, a);

  const auto hq = download<__half>(q), hk = download<__half>(kc), hv = download<__half>(vc);
  double worst_q = 0, worst_k = 0, worst_v = 0;
  for (int i = 0; i < kTokens; ++i)
    for (int h = 0; h < kHeads + kKv; ++h) {
      const auto want = turned(x, i, h, h < kHeads ? gq : gk);
      for (int d = 0; d < kDim; ++d) {
        const size_t at = h < kHeads ? ((size_t)i * kHeads + h) * kDim + d
                                     : ((size_t)i * kKv + h - kHeads) * kDim + d;
        const double e = std::fabs(__half2float(h < kHeads ? hq[at] : hk[at]) - want[d]);
        double& w = h < kHeads ? worst_q : worst_k;
        w = std::fmax(w, e / bound(want[d], 8));
      }
    }
  for (int i = 0; i < kTokens; ++i)
    for (int d = 0; d < kKv * kDim; ++d)
      if (__half2float(hv[(size_t)i * kKv * kDim + d]) !=
          __half2float(x[(size_t)i * kWidth + (kHeads + kKv) * kDim + d]))
        worst_v = 2;
  report("rope q", worst_q);
  report("rope k into a cache", worst_k);
  report("v into a cache", worst_v);

  // causal attention of all tokens over the cache, and of the last one alone
  const std::vector<int32_t> lengths{kTokens};
  DeviceBuffer dlen = upload(lengths);
  for (const int n : {kTokens, 1}) {
    const __half* from = halves(q) + (size_t)(kTokens - n) * kHeads * kDim;
    bbh_attend_args t = attend_args(heads_of(from, kHeads, kDim), heads_of(halves(kc), kKv, kDim),
                                    heads_of(halves(vc), kKv, kDim), heads_of(halves(out), kHeads, kDim),
                                    1, n, kSlots, kHeads, kKv, kDim);
    t.k_lengths = static_cast<const int32_t*>(dlen.data());
    t.right = 0;
    DeviceBuffer scratch(bbh_attend_scratch(&t) + 16);
    t.scratch = scratch.data();
    t.scratch_bytes = scratch.bytes();
    launch_attend(t);
    const auto o = download<__half>(out);
    double worst = 0;
    for (int i = 0; i < n; ++i)
      for (int h = 0; h < kHeads; ++h) {
        const int p = kTokens - n + i, g = h / (kHeads / kKv);
        std::vector<double> s(p + 1);
        double top = -1e300, sum = 0;
        for (int j = 0; j <= p; ++j) {
          s[j] = 0;
          for (int d = 0; d < kDim; ++d)
            s[j] += __half2float(hq[((size_t)p * kHeads + h) * kDim + d]) *
                    (double)__half2float(hk[((size_t)j * kKv + g) * kDim + d]) / 8;
          top = std::fmax(top, s[j]);
        }
        for (int j = 0; j <= p; ++j) sum += s[j] = std::exp(s[j] - top);
        for (int d = 0; d < kDim; ++d) {
          double want = 0;
          for (int j = 0; j <= p; ++j)
            want += s[j] / sum * __half2float(hv[((size_t)j * kKv + g) * kDim + d]);
          const double e = std::fabs(__half2float(o[((size_t)i * kHeads + h) * kDim + d]) - want);
          // weights rounded to fp16 of values up to 2 (2^-10 in all), the output once
          worst = std::fmax(worst, e / (2.0 / 1024 + bound(want, 8)));
        }
      }
    report(n == 1 ? "attention of one token over a cache" : "causal attention", worst);
  }
  std::printf("%d failure(s)\n", failures);
  return failures != 0;
}

// 8-bit rows: quantising, reading back, and the residual norms that quantise
// what they compute.
//
// A row's codes need its largest magnitude first, so the row stays in
// registers between the reductions and its values are read once and written
// once: bound by HBM, at 6.1-6.7 TB/s of those bytes from 100 MB of rows on
// (65536 x 1536 quantised in 49 us and read back in 50; LayerNorm of 131072 x
// 384 with residual and y 56, RMS norm of 16384 x 4096 71), and by a launch and
// its first latency below a few hundred rows (2003 x 384: 2.8-4.1 us).  T
// threads own a row, thread t the 8-wide chunks t, t + T, ..., V of them:
// 16-byte loads, 8-byte stores of codes, any row length and alignment (the last
// chunk of a row goes element by element).
//
// The largest magnitude is reduced on the bit patterns as unsigned integers:
// they order like the magnitudes, an infinity above every number and a NaN
// above that, so one reduction also tells whether the row is finite.

#include <algorithm>

#include "int8.h"

namespace bbh {
namespace {

typedef f16x8 f16x8_any __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

enum Kind { kPlain, kRms, kLayer };

struct UMaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
  }
};

// Reduction over the T threads of a row.  T > 64: over the workgroup, through
// `part` (one array a call: the next call's writes need no barrier before them).
template <int T, class F>
__device__ __forceinline__ float row_reduce(float v, F f, float* part) {
  v = xor_op<8>(v, f);
  v = xor_op<4>(v, f);
  v = xor_op<2>(v, f);
  v = xor_op<1>(v, f);
  if constexpr (T >= 64) {
    v = xor_op<32>(v, f);
    v = xor_op<16>(v, f);
  }
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) v = f(v, part[w]);
  }
  return v;
}

// Chunk `c` of a row of D halves; zeros past the row's end.  STREAM: past the
// caches' reach (streams(), below).
template <bool STREAM = false>
__device__ __forceinline__ f16x8 load8(const f16* row, int c, int D) {
  const int o = c * 8;
  if (o + 8 <= D) {
    const f16x8_any* p = reinterpret_cast<const f16x8_any*>(row + o);
    return STREAM ? __builtin_nontemporal_load(p) : *p;
  }
  f16x8 a;
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = o + e < D ? row[o + e] : (f16)0.f;
  return a;
}

template <bool STREAM>
__device__ __forceinline__ void store8(f16* row, int c, int D, const float (&v)[8]) {
  const int o = c * 8;
  if (o + 8 <= D) {
    f16x8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (f16)v[e];
    f16x8_any* p = reinterpret_cast<f16x8_any*>(row + o);
    if constexpr (STREAM)
      __builtin_nontemporal_store(a, p);
    else
      *p = a;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (o + e < D) row[o + e] = (f16)v[e];
  }
}

// How a row's values become codes: v / scale = 127 v / amax.
struct Coder {
  float amax, inv;
  bool finite;
  // (Below 2^-120, which no fp16 row reaches, the reciprocal would overflow.)
  __device__ __forceinline__ explicit Coder(float a) : amax(a) {
    finite = __float_as_uint(amax) < 0x7f800000u;
    inv = finite && amax >= 0x1p-120f ? 1.0f / amax : 0.f;
  }
  __device__ __forceinline__ float scale() const {
    return finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
  }
  // The rounded code in the low byte.  The product with the reciprocal is off
  // by up to 2^-16 of a step near 127, enough to push an exact tie to the wrong
  // side; one correction by its remainder gives the quotient rounded once.
  // (127 v is exact for v from fp16.)  Adding 1.5 * 2^23 rounds to an integer,
  // ties to even, and leaves it in two's complement in the sum's low bits.
  __device__ __forceinline__ uint32_t code(float v) const {
    const float t = 127.0f * v, q = t * inv;
    const float c = fmaf(fmaf(-q, amax, t), inv, q);
    return __float_as_uint(c + 12582912.0f);
  }
  __device__ __forceinline__ uint32_t code4(const float* v) const {
    // perm selects bytes of {a, b}: 0-3 from b, 4-7 from a
    const uint32_t lo = __builtin_amdgcn_perm(code(v[1]), code(v[0]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(code(v[3]), code(v[2]), 0x04000c0cu);
    return finite ? lo | hi : 0u;
  }
};

__device__ __forceinline__ void store_codes(int8_t* row, int c, int D, const Coder& k,
                                            const float (&v)[8]) {
  const int o = c * 8;
  const u32x2 w = {k.code4(v), k.code4(v + 4)};
  if (o + 8 <= D) {
    *reinterpret_cast<u32x2_any*>(row + o) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (o + e < D) row[o + e] = (int8_t)(w[e / 4] >> (8 * (e % 4)));
  }
}

// This workgroup's first row (or item) of a launch of grid2().
__device__ __forceinline__ int64_t block_id() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

struct NormArgs {
  const f16 *residual, *gamma, *beta;
  f16 *sum, *y;
  float eps;
};

// x and the outputs may be the same rows, so none is __restrict__; every
// thread writes only the elements it has read.
template <int T, int V, Kind KIND, bool STREAM>
__global__ __launch_bounds__(T < 256 ? 256 : T) void quantize_kernel(const f16* x, int8_t* q,
                                                                     float* scale, int M, int D,
                                                                     NormArgs a) {
  constexpr int R = T < 256 ? 256 / T : 1;  // rows a workgroup
  __shared__ float part[4][T > 64 ? T / 64 : 1];
  const int64_t row = block_id() * R + threadIdx.x / T;
  const int t = threadIdx.x % T;
  if (row >= M) return;  // T > 64: the whole workgroup
  const size_t off = (size_t)row * D;
  const int chunks = (D + 7) / 8;
  // Every load before the first use: x, the residual and the norm's weights
  // come in one latency.
  f16x8 hx[V], hr[V], hg[V], hb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    hx[i] = f16x8{};
    if (t + T * i < chunks) hx[i] = load8<STREAM>(x + off, t + T * i, D);
  }
  if constexpr (KIND != kPlain) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      hr[i] = f16x8{};
      if (a.residual && t + T * i < chunks) hr[i] = load8<STREAM>(a.residual + off, t + T * i, D);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      hg[i] = hb[i] = f16x8{};
      if (t + T * i < chunks) {
        hg[i] = load8(a.gamma, t + T * i, D);
        if constexpr (KIND == kLayer) hb[i] = load8(a.beta, t + T * i, D);
      }
    }
  }
  float v[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[i][e] = (float)hx[i][e];
      if constexpr (KIND != kPlain) v[i][e] += (float)hr[i][e];
    }
  if constexpr (KIND != kPlain) {
    if (a.sum) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (t + T * i < chunks) store8<STREAM>(a.sum + off, t + T * i, D, v[i]);
    }
    if constexpr (KIND == kLayer) {
      // Twice: the mean of rows of nearly equal values is off by more than they
      // deviate (a rounded sum), so the deviations' own mean comes off them too.
      // Of equal values nothing is left then: the deviations are a few steps of
      // fp32, all alike, and their sum and its quotient exact.
      // (1 x 384 2.3 us with one mean, 2.4 with both; 8192 x 384 8.2 either way,
      // 131072 x 32 15.4 and 16.1.)
#pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) s += v[i][e];
        const float mean = row_reduce<T>(s, AddOp{}, part[pass]) / (float)D;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int n = D - (t + T * i) * 8;  // values of this chunk
          if (n >= 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] -= mean;
          } else if (n > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] -= e < n ? mean : 0.f;
          }
        }
      }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[i][e] * v[i][e];
    const float rstd = rsqrtf(row_reduce<T>(s, AddOp{}, part[2]) / (float)D + a.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = v[i][e] * rstd * (float)hg[i][e];
        if constexpr (KIND == kLayer) v[i][e] += (float)hb[i][e];
      }
      if (a.y && t + T * i < chunks) store8<STREAM>(a.y + off, t + T * i, D, v[i]);
    }
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = UMaxOp{}(m, fabsf(v[i][e]));
  const Coder k(row_reduce<T>(m, UMaxOp{}, part[3]));
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = t + T * i;
    if (c < chunks) store_codes(q + off, c, D, k, v[i]);
  }
  if (t == 0) scale[row] = k.scale();
}

// Rows longer than 16384: one workgroup a row, read twice (the second time
// from L2).
constexpr int kWide = 1024;
__global__ __launch_bounds__(kWide) void quantize_wide_kernel(const f16* __restrict__ x,
                                                              int8_t* __restrict__ q,
                                                              float* __restrict__ scale, int M,
                                                              int D) {
  __shared__ float part[kWide / 64];
  const int64_t row = block_id();
  if (row >= M) return;
  const size_t off = (size_t)row * D;
  const int chunks = (D + 7) / 8;
  float m = 0.f;
  for (int c = threadIdx.x; c < chunks; c += kWide) {
    const f16x8 h = load8(x + off, c, D);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = UMaxOp{}(m, fabsf((float)h[e]));
  }
  const Coder k(row_reduce<kWide>(m, UMaxOp{}, part));
  for (int c = threadIdx.x; c < chunks; c += kWide) {
    const f16x8 h = load8(x + off, c, D);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
    store_codes(q + off, c, D, k, v);
  }
  if (threadIdx.x == 0) scale[row] = k.scale();
}

// T threads a row, eight codes at a time.
template <int T, bool STREAM>
__global__ __launch_bounds__(256) void dequantize_kernel(const int8_t* __restrict__ q,
                                                         const float* __restrict__ scale,
                                                         f16* __restrict__ x, int M, int D) {
  const int64_t row = block_id() * (256 / T) + threadIdx.x / T;
  if (row >= M) return;
  const size_t off = (size_t)row * D;
  const float s = scale[row];
  for (int c = threadIdx.x % T; c < (D + 7) / 8; c += T) {
    const int o = c * 8;
    float v[8];
    if (o + 8 <= D) {
      const u32x2 w = *reinterpret_cast<const u32x2_any*>(q + off + o);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * s;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = o + e < D ? (float)q[off + o + e] * s : 0.f;
    }
    store8<STREAM>(x + off, c, D, v);
  }
}

// n workgroups: no launch dimension counts 2^32 threads.
dim3 grid2(int64_t n) {
  constexpr int64_t X = 1 << 21;
  return n <= X ? dim3((uint32_t)n) : dim3((uint32_t)X, (uint32_t)((n + X - 1) / X));
}

template <int T, bool STREAM>
hipError_t dequantize(const int8_t* q, const float* scale, f16* x, int M, int D, hipStream_t s) {
  constexpr int R = 256 / T;
  hipLaunchKernelGGL((dequantize_kernel<T, STREAM>), grid2(((int64_t)M + R - 1) / R), dim3(256), 0, s, q,
                     scale, x, M, D);
  return hipGetLastError();
}

template <int T, int V, Kind KIND, bool STREAM>
hipError_t launch(const f16* x, int8_t* q, float* scale, int M, int D, const NormArgs& a,
                  hipStream_t s) {
  constexpr int R = T < 256 ? 256 / T : 1;
  hipLaunchKernelGGL((quantize_kernel<T, V, KIND, STREAM>), grid2(((int64_t)M + R - 1) / R),
                     dim3(T < 256 ? 256 : T), 0, s, x, q, scale, M, D, a);
  return hipGetLastError();
}

template <Kind KIND, bool STREAM>
hipError_t quantize_as(const f16* x, int8_t* q, float* scale, int M, int D, const NormArgs& a,
                       hipStream_t s) {
  // Threads a row: as few as leave a thread at most four chunks, so that the
  // lanes are full and the reductions short; more where rows are too few to fill
  // the GPU and a thread's chunks would queue behind each other.  Measured, us
  // (quantise / LayerNorm with residual and y; inputs that change from call to
  // call):
  //   131072 x 32     16 threads  8.3 / 16.5   64 threads  25.9 / 56.0
  //   2003 x 384      16 x 3      3.1 /  4.8   64 x 1       2.8 /  4.1
  //   4096 x 384      16 x 3      3.5 /  5.5   64 x 1       3.5 /  5.5
  //   8192 x 384      16 x 3      4.3 /  7.5   64 x 1       4.4 /  7.9
  //   32768 x 384     16 x 3      9.8 / 20.3   64 x 1      11.5 / 20.8
  //   131072 x 384    16 x 3     26.7 / 55.9   64 x 1      34.5 / 69.4
  //   2048 x 256      16 x 2      2.7 /  3.8   64 x 1       2.7 /  3.6
  //   4096 x 256      16 x 2      2.8 /  4.5   64 x 1       3.1 /  5.2
  //   30000 x 512     16 x 4     11.9 / 23.9   64 x 1      12.0 / 22.1
  //   131072 x 512    16 x 4     34.2 / 74.1   64 x 1      38.0 / 74.9
  //   700 x 2048      64 x 4      3.6 /  5.8   256 x 1      3.3 /  5.3
  //   5000 x 1700     64 x 4      9.1 / 21.3   256 x 1      9.0 / 22.4
  //   65536 x 1536    64 x 3     48.8 / 105    256 x 1     64.7 / 137
  //   65536 x 1792    64 x 4     57.7 / 126    256 x 1     70.1 / 146
  //   1 x 8192       256 x 4      3.0 /  5.2   1024 x 1     2.7 /  4.3
  //   100 x 8192     256 x 4      3.4 /  6.0   1024 x 1     3.0 /  5.3
  //   2048 x 8192    256 x 4     13.0 / 26.6   1024 x 1    14.0 / 28.4
  //   8192 x 8192    256 x 4     34.5 / 78.5   1024 x 1    43.7 / 93.7
  const int chunks = (D + 7) / 8;
  const bool many = M >= 4096;
  if (chunks <= 16) return launch<16, 1, KIND, STREAM>(x, q, scale, M, D, a, s);
  if (chunks <= 32 && many) return launch<16, 2, KIND, STREAM>(x, q, scale, M, D, a, s);
  if (chunks <= 48 && many) return launch<16, 3, KIND, STREAM>(x, q, scale, M, D, a, s);
  if constexpr (STREAM) {
    if (chunks <= 64) return launch<16, 4, KIND, true>(x, q, scale, M, D, a, s);
  } else {
    if (chunks <= 64) return launch<64, 1, KIND, false>(x, q, scale, M, D, a, s);
  }
  if (chunks <= 128) return launch<64, 2, KIND, STREAM>(x, q, scale, M, D, a, s);
  if (chunks <= 192) return launch<64, 3, KIND, STREAM>(x, q, scale, M, D, a, s);
  if constexpr (STREAM) {
    if (chunks <= 256) return launch<64, 4, KIND, true>(x, q, scale, M, D, a, s);
  } else {
    if (chunks <= 256) return launch<256, 1, KIND, false>(x, q, scale, M, D, a, s);
    if (chunks > 512 && chunks <= 1024 && M <= 128)
      return launch<1024, 1, KIND, false>(x, q, scale, M, D, a, s);
  }
  if (chunks <= 512) return launch<256, 2, KIND, STREAM>(x, q, scale, M, D, a, s);
  if (chunks <= 768) return launch<256, 3, KIND, STREAM>(x, q, scale, M, D, a, s);
  if (chunks <= 1024) return launch<256, 4, KIND, STREAM>(x, q, scale, M, D, a, s);
  return launch<1024, 2, KIND, STREAM>(x, q, scale, M, D, a, s);
}

// fp16 rows of this many bytes and more are read and written past the caches
// (non-temporal): they would push out of the memory-side cache what the next
// operators find there, the codes among it, and be gone themselves before anyone
// came back to them.  Quantising and reading back 131072 x 384 (96 MB) 54.5 us
// without, 49.4 with; LayerNorm with residual and y 64.0 and 55.9, of 65536 x 384 34.5
// and 30.5.  Inputs that the call before read are the other side: 47.2 and 49.6,
// 62.4 and 56.2, 28.5 and 30.0; 20.1 and 23.9 for quantising and reading back 43690 x
// 384 (32 MB), so smaller ones stay in the caches.  (Rows of 63, whose lines are
// shared: LayerNorm of 400003 93.5 and 98.0, 68.3 and 96.8.)  Values read back stay
// up to twice the size.
constexpr int64_t kStreamBytes = 48 << 20;
bool streams(int M, int D, int64_t bytes) { return (int64_t)M * D * 2 >= bytes; }

template <Kind KIND>
hipError_t quantize(const f16* x, int8_t* q, float* scale, int M, int D, const NormArgs& a,
                    hipStream_t s) {
  return streams(M, D, kStreamBytes) ? quantize_as<KIND, true>(x, q, scale, M, D, a, s)
                                     : quantize_as<KIND, false>(x, q, scale, M, D, a, s);
}

template <bool STREAM>
hipError_t dequantize_as(const int8_t* q, const float* scale, f16* x, int M, int D,
                         hipStream_t s) {
  // 131072 x 256 18.9 us with 16 threads a row, 25.5 with 64; 65536 x 1024 31.2
  // and 29.8; 700 x 2048 3.3 with 64, 2.7 with 256, 16384 x 4096 31.5 and 29.4
  if (D <= 256) return dequantize<16, STREAM>(q, scale, x, M, D, s);
  if (D <= 1024) return dequantize<64, STREAM>(q, scale, x, M, D, s);
  return dequantize<256, STREAM>(q, scale, x, M, D, s);
}

}  // namespace

hipError_t quantize_rows(const f16* x, int8_t* q, float* scale, int M, int D, hipStream_t s) {
  if (D <= kMaxNormRow) return quantize<kPlain>(x, q, scale, M, D, NormArgs{}, s);
  hipLaunchKernelGGL(quantize_wide_kernel, grid2(M), dim3(kWide), 0, s, x, q, scale, M, D);
  return hipGetLastError();
}

hipError_t dequantize_rows(const int8_t* q, const float* scale, f16* x, int M, int D,
                           hipStream_t s) {
  return streams(M, D, 2 * kStreamBytes) ? dequantize_as<true>(q, scale, x, M, D, s)
                                         : dequantize_as<false>(q, scale, x, M, D, s);
}

hipError_t rmsnorm_quantize(const f16* x, const f16* residual, const f16* gamma, f16* sum, f16* y,
                            int8_t* q, float* scale, int M, int D, float eps, hipStream_t s) {
  return quantize<kRms>(x, q, scale, M, D, NormArgs{residual, gamma, nullptr, sum, y, eps}, s);
}

hipError_t layernorm_quantize(const f16* x, const f16* residual, const f16* gamma,
                              const f16* beta, f16* sum, f16* y, int8_t* q, float* scale, int M,
                              int D, float eps, hipStream_t s) {
  return quantize<kLayer>(x, q, scale, M, D, NormArgs{residual, gamma, beta, sum, y, eps}, s);
}

}  // namespace bbh

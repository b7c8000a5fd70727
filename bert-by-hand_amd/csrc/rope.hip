// Heads normed and rotated by their positions, out of fused QKV rows or over them,
// keys and values into the slots of a cache where asked: one pass, bound by the
// bytes of the heads (4 an element).
//
// Angles.  Pair i turns by t = position * f_i.  What sin and cos need is t modulo
// a turn, and in floating point a far position leaves few digits of that (position
// 10^6 at f = 1: 0.06 radians in fp32).  So a pair's turns a position are a 64-bit
// fixed-point fraction, computed once from the frequency in double: the low 64 bits of
// its product with the position are the fraction of a turn without any loss, and the
// high word of them is off by less than 2^-31 turns for every int32 position.
//
// A workgroup takes some whole rows (or a part of the heads of one, where rows are few):
// its threads compute the sines and cosines of the rows' pairs into LDS while the first
// heads are on their way, then every thread turns its pieces of heads.
#include <algorithm>

#include "attend.h"

namespace bbh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;

// (cos, sin), times the magnitude, of pair i at a position.
__device__ __forceinline__ float2 angle(const RopeParams& p, const RopeSteps& steps, int position,
                                        int i) {
  const uint2 st = steps.step[i];
  const uint32_t at = (uint32_t)position;
  // high word of (int64)position * step
  uint32_t turn = __umulhi(at, st.x) + at * st.y;
  if (position < 0) turn -= st.x;
  float s, c;
  sincospif((float)(int32_t)turn * 0x1p-31f, &s, &c);  // half turns
  return make_float2(c * p.magnitude, s * p.magnitude);
}
__device__ __forceinline__ int position_of(const RopeParams& p, int row) {
  return p.rot == 0 ? 0 : p.positions ? p.positions[row] : row % p.seq;
}

__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
  const float a0 = a;
  a = a0 * cs.x - b * cs.y;
  b = b * cs.x + a0 * cs.y;
}

// Sum over groups of G neighbouring lanes.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (G >= 2) v = xor_op<1>(v, AddOp{});
  if constexpr (G >= 4) v = xor_op<2>(v, AddOp{});
  if constexpr (G >= 8) v = xor_op<4>(v, AddOp{});
  if constexpr (G >= 16) v = xor_op<8>(v, AddOp{});
  if constexpr (G >= 32) v = xor_op<16>(v, AddOp{});
  if constexpr (G >= 64) v = xor_op<32>(v, AddOp{});
  return v;
}

template <int W>
using Half = _Float16 __attribute__((ext_vector_type(W)));

template <bool STREAM, class V>
__device__ __forceinline__ V take(const f16* p) {
  const V* v = reinterpret_cast<const V*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(v);
  return *v;
}
template <bool STREAM, class V>
__device__ __forceinline__ void put(f16* p, V v) {
  V* o = reinterpret_cast<V*>(p);
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, o);
  else
    *o = v;
}

// How a launch is cut: pieces of 2 W values (`units` a head), U a thread.
struct Cut {
  int rows, parts;  // rows of a workgroup; workgroups a row's heads are spread over
  int units, unit_div, head_div;  // division by units and heads: (n * div) >> 20, n < 1024
};

// A piece is two runs of W values: the same place in both halves of the turning part, or
// neighbours (interleaved pairs, and the values that do not turn).  G: lanes a head, a power
// of two, where heads are normed (their squares are added across lanes); 0: as many as it has
// pieces.
template <int W, int G, int U, bool STREAM>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams p, RopeSteps steps, Cut cut) {
  constexpr bool NORM = G > 0;
  using V = Half<W>;
  HIP_DYNAMIC_SHARED(float2, cs);  // [rows][rot / 2]
  __shared__ f16 gammas[NORM ? 2 : 1][NORM ? 2 * kMaxRopePairs : 1];
  const int tid = threadIdx.x;
  const int block = blockIdx.x / cut.parts, part = blockIdx.x - block * cut.parts;
  const int r0 = p.row0 + block * cut.rows, rows = min(cut.rows, p.rows - r0);
  const int heads = p.q.heads + p.k.heads + p.v.heads, lanes = NORM ? G : cut.units;
  const V none = {};

  struct At {
    const f16* x;
    f16* y;
    int kind, u, row;  // kind 0 q, 1 k, 2 v, 3 nothing; row of the workgroup's
  };
  auto locate = [&](int n) {  // piece n of this thread
    const int i = tid + n * kThreads;
    const int hs = NORM ? i / (G ? G : 1) : (i * cut.unit_div) >> 20;
    At a{nullptr, nullptr, 3, i - hs * lanes, 0};
    int h = hs;
    if (cut.parts > 1) {
      h += part * (U * kThreads / lanes);
      if (hs >= U * kThreads / lanes) h = heads;
    } else {
      a.row = (hs * cut.head_div) >> 20;
      h -= a.row * heads;
      if (a.row >= rows) h = heads;
    }
    const int row = r0 + a.row;
    if (h >= heads) a.row = 0;
    if (h < p.q.heads) {
      a.x = p.q.x + row * p.q.x_row + h * p.q.x_head;
      a.y = p.q.y + row * p.q.y_row + h * p.q.y_head;
      a.kind = 0;
    } else if (h < heads) {
      h -= p.q.heads;
      const bool k = h < p.k.heads;
      const RopeParams::Part& t = k ? p.k : p.v;
      if (!k) h -= p.k.heads;
      const int64_t to = p.kv_rows ? p.kv_rows[row] : row;
      if (!p.kv_rows || (to >= 0 && to < p.kv_out_rows)) {
        a.x = t.x + row * t.x_row + h * t.x_head;
        a.y = t.y + to * t.y_row + h * t.y_head;
        a.kind = k ? 1 : 2;
      }
    }
    return a;
  };
  At at[U];
  V a[U], b[U];
  auto place = [&](int u, int& ca, int& cb) {  // first values of a piece's runs
    const bool half = !p.interleaved && 2 * W * u < p.rot;
    ca = half ? W * u : 2 * W * u;
    cb = half ? ca + p.rot / 2 : ca + W;
  };
#pragma unroll
  for (int e = 0; e < U; ++e) {
    at[e] = locate(e);
    int ca, cb;
    place(at[e].u, ca, cb);
    a[e] = b[e] = none;
    if (at[e].kind < 3 && ca < p.dim) a[e] = take<STREAM, V>(at[e].x + ca);
    if (at[e].kind < 3 && cb < p.dim) b[e] = take<STREAM, V>(at[e].x + cb);
  }
  if constexpr (NORM) {
    if (tid < p.dim) {
      if (p.q.gamma) gammas[0][tid] = p.q.gamma[tid];
      if (p.k.gamma) gammas[1][tid] = p.k.gamma[tid];
    }
  }
  const int pairs = p.rot / 2;
  for (int i = tid; i < rows * pairs; i += kThreads) {
    const int r = i / pairs;
    cs[i] = angle(p, steps, position_of(p, r0 + r), i - r * pairs);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < U; ++e) {
    const int kind = at[e].kind, u = at[e].u;
    int ca, cb;
    place(u, ca, cb);
    V oa = a[e], ob = b[e];
    float x[W], y[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      x[i] = (float)oa[i];
      y[i] = (float)ob[i];
    }
    bool changed = false;
    if constexpr (NORM) {
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) q = fmaf(x[i], x[i], fmaf(y[i], y[i], q));
      q = lanes_sum<G>(q);
      changed = kind == 0 ? p.q.gamma != nullptr : kind == 1 && p.k.gamma != nullptr;
      if (changed) {
        const float r = rsqrtf(q / (float)p.dim + p.eps);
        const f16* g = gammas[kind];
#pragma unroll
        for (int i = 0; i < W; ++i) {
          x[i] *= r * (float)g[min(ca, p.dim - W) + i];
          y[i] *= r * (float)g[min(cb, p.dim - W) + i];
        }
      }
    }
    if (kind < 2 && 2 * W * u < p.rot) {
      changed = true;
      const float2* t = cs + at[e].row * pairs + W * u;
      float2 v[W];
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = t[i];
      if (p.interleaved) {  // pairs (x0, x1), (x2, x3), ... (y0, y1), ...
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          turn(x[2 * i], x[2 * i + 1], v[i]);
          turn(y[2 * i], y[2 * i + 1], v[W / 2 + i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) turn(x[i], y[i], v[i]);
      }
    }
    if (changed) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        oa[i] = (f16)x[i];
        ob[i] = (f16)y[i];
      }
    }
    if (kind < 3 && ca < p.dim) put<STREAM>(at[e].y + ca, oa);
    if (kind < 3 && cb < p.dim) put<STREAM>(at[e].y + cb, ob);
  }
}

// Any sizes and alignment: a wavefront for the heads of a row, one after another, an element or a
// pair a lane.  Bound by the number of accesses of 2 bytes (32768 rows of 16 heads of 65 values 93
// us, 1.5 TB/s; 24 of 127 158 us, 2.5 TB/s).
__global__ __launch_bounds__(64 * kWaves) void rope_any_kernel(RopeParams p, RopeSteps steps) {
  __shared__ float2 lds[kWaves][kMaxRopePairs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kWaves + wave;
  const int row = p.row0 + (int)w;
  if (row >= p.rows) return;
  int64_t out_row = row;
  if (p.kv_rows) out_row = p.kv_rows[row];
  const bool kv_on = !p.kv_rows || (out_row >= 0 && out_row < p.kv_out_rows);
  const int position = position_of(p, row);
  float2* cs = lds[wave];
  for (int i = lane; 2 * i < p.rot; i += kWave) cs[i] = angle(p, steps, position, i);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const int pairs = p.rot / 2;
  auto heads = [&](const RopeParams::Part& t, int64_t yr, bool turns) {
    for (int h = 0; h < t.heads; ++h) {
      const f16* x = t.x + row * t.x_row + h * t.x_head;
      f16* y = t.y + yr * t.y_row + h * t.y_head;
      if (!turns) {
        for (int d = lane; d < p.dim; d += kWave) y[d] = x[d];
        continue;
      }
      float pa[2] = {}, pb[2] = {};
      f16 rest[4] = {};  // (as they are: a conversion and back makes a signalling NaN a quiet one)
      float q = 0.f;
      auto index = [&](int i, int which) {
        return p.interleaved ? 2 * i + which : i + which * pairs;
      };
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = lane + 64 * e;
        if (i < pairs) {
          pa[e] = (float)x[index(i, 0)];
          pb[e] = (float)x[index(i, 1)];
          q = fmaf(pa[e], pa[e], fmaf(pb[e], pb[e], q));
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = p.rot + lane + 64 * e;
        if (d < p.dim) {
          rest[e] = x[d];
          q = fmaf((float)rest[e], (float)rest[e], q);
        }
      }
      const bool norm = t.gamma != nullptr;
      float r = 1.f;
      if (norm) r = rsqrtf(wave_sum(q) / (float)p.dim + p.eps);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = lane + 64 * e;
        if (i < pairs) {
          const int ia = index(i, 0), ib = index(i, 1);
          float u = pa[e], v = pb[e];
          if (norm) {
            u *= r * (float)t.gamma[ia];
            v *= r * (float)t.gamma[ib];
          }
          turn(u, v, cs[i]);
          y[ia] = (f16)u;
          y[ib] = (f16)v;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = p.rot + lane + 64 * e;
        if (d < p.dim) y[d] = norm ? (f16)((float)rest[e] * (r * (float)t.gamma[d])) : rest[e];
      }
    }
  };
  heads(p.q, row, true);
  if (kv_on) {
    heads(p.k, out_row, true);
    heads(p.v, out_row, false);
  }
}

// Values that every address and stride of a part allows to be moved at once.
int width(const RopeParams::Part& t, int w) {
  if (!t.heads) return w;
  const uint64_t all = ((uint64_t)(uintptr_t)t.x | (uint64_t)(uintptr_t)t.y) / 2 |
                       (uint64_t)(t.x_row | t.x_head | t.y_row | t.y_head);
  while (w > 1 && (all & (w - 1))) w /= 2;
  return ((uintptr_t)t.x | (uintptr_t)t.y) & 1 ? 1 : w;
}

// Whether rows are read and written past the caches: from 48 MB on, where every store is of whole
// lines (131072 x 24 x 32, whose stores are of half lines, 81 -> 139 us), with three pieces a thread
// where heads are normed, two otherwise.  40 heads of 128, us with two pieces through the caches /
// past them with two, three, four:
//   normed      32 MB 17.3 / 17.5, 16.8, 19.3   48: 27.2 / 23.8, 21.7, 22.4   320: 141 / 135, 129, 132
//   not normed  32 MB 12.9 / 13.7, 15.1, 16.6   48: 20.3 / 19.0, 20.6, 21.3   320: 117 / 105, 111, 119
constexpr int64_t kStreamBytes = 48 << 20;
bool lines(const RopeParams::Part& t) {
  return !t.heads || (((uintptr_t)t.y & 127) == 0 && ((t.y_row | t.y_head) & 63) == 0);
}
bool streams(const RopeParams& p) {
  const int64_t bytes = 2 * (int64_t)(p.rows - p.row0) * (p.q.heads + p.k.heads + p.v.heads) * p.dim;
  return bytes >= kStreamBytes && !p.interleaved && p.rot == p.dim && p.dim % 128 == 0 && lines(p.q) &&
         lines(p.k) && lines(p.v);
}

int pow2(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

template <int W, int G, int U, bool STREAM>
hipError_t launch_as(const RopeParams& p, const RopeSteps& steps, hipStream_t s) {
  const int heads = p.q.heads + p.k.heads + p.v.heads;
  Cut c{};
  c.units = (p.dim + 2 * W - 1) / (2 * W);
  const int lanes = G ? G : c.units, at_once = U * kThreads / lanes;  // heads of a workgroup
  c.rows = std::max(1, std::min(at_once / heads, 2048 / std::max(1, p.rot / 2)));
  c.parts = (heads + at_once - 1) / at_once;
  c.unit_div = ((1 << 20) + c.units - 1) / c.units;
  c.head_div = ((1 << 20) + heads - 1) / heads;
  const int rows = p.rows - p.row0;
  const int64_t grid = (int64_t)((rows + c.rows - 1) / c.rows) * c.parts;
  const size_t lds = (size_t)c.rows * (p.rot / 2) * sizeof(float2);
  hipLaunchKernelGGL((rope_kernel<W, G, U, STREAM>), dim3((unsigned)grid), dim3(kThreads), lds, s, p, steps, c);
  return hipGetLastError();
}
template <int W, int G>
hipError_t launch(const RopeParams& p, const RopeSteps& steps, hipStream_t s) {
  const int64_t items = (int64_t)(p.rows - p.row0) * (p.q.heads + p.k.heads + p.v.heads) *
                        (G ? G : (p.dim + 2 * W - 1) / (2 * W));
  // A piece a thread for calls of few tokens (16 tokens of 48 heads of 128: 4.0 us against 5.5 with
  // four), two otherwise (131072 x 24 x 32 81 us with two, 93 with four).
  if (items < 1 << 18) return launch_as<W, G, 1, false>(p, steps, s);
  if constexpr (W == 8) {
    if (streams(p)) return launch_as<W, G, G ? 3 : 2, true>(p, steps, s);
  }
  return launch_as<W, G, 2, false>(p, steps, s);
}
template <int W>
hipError_t launch_w(const RopeParams& p, const RopeSteps& steps, hipStream_t s) {
  if (!p.q.gamma && !p.k.gamma) return launch<W, 0>(p, steps, s);
  const int g = pow2((p.dim + 2 * W - 1) / (2 * W));
  if constexpr (W <= 2) {
    if (g > 32) return launch<W, 64>(p, steps, s);
  }
  if constexpr (W <= 4) {
    if (g > 16) return launch<W, 32>(p, steps, s);
  }
  return g > 8 ? launch<W, 16>(p, steps, s)
         : g > 4 ? launch<W, 8>(p, steps, s)
         : g > 2 ? launch<W, 4>(p, steps, s)
         : g > 1 ? launch<W, 2>(p, steps, s)
                 : launch<W, 1>(p, steps, s);
}

}  // namespace

hipError_t rope_heads(const RopeParams& args, const RopeSteps& steps, hipStream_t s) {
  // values moved at once: what addresses, strides, the head and the turning part allow
  int w = width(args.v, width(args.k, width(args.q, 8)));
  while (w > 1 && (args.dim % w || args.rot % (2 * w))) w /= 2;
  const int heads = args.q.heads + args.k.heads + args.v.heads;
  // rows of a launch: threads are counted in 32 bits, and 64 * heads cover a row's
  const int most = std::max(1, (1 << 30) / (64 * heads + kThreads));
  for (int row0 = 0; row0 < args.rows;) {
    RopeParams p = args;
    const int rows = std::min(most, args.rows - row0);
    p.row0 = row0;
    p.rows = row0 + rows;
    hipError_t e;
    if (w == 1) {
      hipLaunchKernelGGL(rope_any_kernel, dim3((unsigned)((rows + kWaves - 1) / kWaves)),
                         dim3(kThreads), 0, s, p, steps);
      e = hipGetLastError();
    } else {
      e = w == 8   ? launch_w<8>(p, steps, s)
          : w == 4 ? launch_w<4>(p, steps, s)
                   : launch_w<2>(p, steps, s);
    }
    if (e != hipSuccess) return e;
    row0 += rows;
  }
  return hipSuccess;
}

}  // namespace bbh

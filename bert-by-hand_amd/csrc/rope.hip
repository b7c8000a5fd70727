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
// A wavefront takes a row.  Its lanes compute the sines and cosines of the row's
// pairs once (one or two a lane), pass them through LDS, and every group of lanes
// then walks heads with them in registers.
#include <algorithm>

#include "attend.h"

namespace bbh {
namespace {

constexpr int kWaves = 4;  // a workgroup

// (cos, sin) of the row's pairs, times the magnitude, into this wavefront's part of LDS.
__device__ __forceinline__ void angles(const RopeParams& p, const RopeSteps& steps, int position,
                                       float2* cs, int lane) {
  for (int i = lane; 2 * i < p.rot; i += kWave) {
    const uint2 st = steps.step[i];
    const uint32_t at = (uint32_t)position;
    // high word of (int64)position * step
    uint32_t turn = __umulhi(at, st.x) + at * st.y;
    if (position < 0) turn -= st.x;
    float s, c;
    sincospif((float)(int32_t)turn * 0x1p-31f, &s, &c);  // half turns
    cs[i] = make_float2(c * p.magnitude, s * p.magnitude);
  }
}

// Sum over groups of G neighbouring lanes.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (G >= 2) v = xor_op<1>(v, AddOp{});
  if constexpr (G >= 4) v = xor_op<2>(v, AddOp{});
  if constexpr (G >= 8) v = xor_op<4>(v, AddOp{});
  if constexpr (G >= 16) v = xor_op<8>(v, AddOp{});
  return v;
}

// G lanes a head, 16 values (two chunks of eight) a lane: in the half layout the
// chunks of a lane hold the two halves of eight pairs, otherwise they are neighbours.
template <int G, bool NORM>
__global__ __launch_bounds__(64 * kWaves) void rope_kernel(RopeParams p, RopeSteps steps, int waves) {
  constexpr int HW = kWave / G, U = 4;  // heads a wavefront takes at once; steps in flight
  __shared__ float2 lds[kWaves][kMaxRopePairs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kWaves + wave;
  const int64_t rw = w / waves;
  const int row = p.row0 + (int)rw, part = (int)(w - rw * waves);
  if (row >= p.rows) return;
  const int u = lane % G, first = part * HW + lane / G, step = waves * HW;
  const int heads = p.q.heads + p.k.heads + p.v.heads;
  int64_t out_row = row;
  if (p.kv_rows) out_row = p.kv_rows[row];
  const bool kv_on = !p.kv_rows || (out_row >= 0 && out_row < p.kv_out_rows);
  const int position = p.rot == 0 ? 0 : p.positions ? p.positions[row] : row % p.seq;

  const bool turns = 16 * u < p.rot, half = turns && !p.interleaved;
  const int ca = half ? 8 * u : 16 * u, cb = half ? ca + p.rot / 2 : ca + 8;
  const bool has_a = ca < p.dim, has_b = cb < p.dim;
  const f16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
  struct At {
    const f16* x;
    f16* y;
    int kind;  // 0 q, 1 k, 2 v, 3 nothing
  };
  auto locate = [&](int h) {
    At a{nullptr, nullptr, 3};
    if (h < p.q.heads) {
      a = {p.q.x + row * p.q.x_row + h * p.q.x_head, p.q.y + row * p.q.y_row + h * p.q.y_head, 0};
    } else if (h < heads && kv_on) {
      h -= p.q.heads;
      const bool k = h < p.k.heads;
      const RopeParams::Part& t = k ? p.k : p.v;
      if (!k) h -= p.k.heads;
      a = {t.x + row * t.x_row + h * t.x_head, t.y + out_row * t.y_row + h * t.y_head, k ? 1 : 2};
    }
    return a;
  };
  At at[U];
  f16x8 a[U], b[U];
  auto load = [&](int h0) {
#pragma unroll
    for (int e = 0; e < U; ++e) {
      at[e] = locate(h0 + e * step);
      a[e] = b[e] = none;
      if (at[e].kind < 3 && has_a) a[e] = *reinterpret_cast<const f16x8*>(at[e].x + ca);
      if (at[e].kind < 3 && has_b) b[e] = *reinterpret_cast<const f16x8*>(at[e].x + cb);
    }
  };
  load(first);
  f16x8 ga[2], gb[2];
  if constexpr (NORM) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const f16* g = e == 0 ? p.q.gamma : p.k.gamma;
      ga[e] = gb[e] = none;
      if (g && has_a)
#pragma unroll
        for (int i = 0; i < 8; ++i) ga[e][i] = g[ca + i];
      if (g && has_b)
#pragma unroll
        for (int i = 0; i < 8; ++i) gb[e][i] = g[cb + i];
    }
  }
  float2* cs = lds[wave];
  angles(p, steps, position, cs, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wavefront's own writes
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = turns ? cs[8 * u + i] : make_float2(1.f, 0.f);
    c[i] = v.x;
    s[i] = v.y;
  }
  for (int h0 = first; h0 - lane / G < heads; h0 += U * step) {
    if (h0 != first) load(h0);
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (at[e].kind > 1) {  // moved as it is, or nothing
        if (at[e].kind == 2 && has_a) *reinterpret_cast<f16x8*>(at[e].y + ca) = a[e];
        if (at[e].kind == 2 && has_b) *reinterpret_cast<f16x8*>(at[e].y + cb) = b[e];
      }
      float x[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = (float)a[e][i];
        y[i] = (float)b[e][i];
      }
      if constexpr (NORM) {
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) q = fmaf(x[i], x[i], fmaf(y[i], y[i], q));
        q = lanes_sum<G>(q);
        const bool k = at[e].kind == 1;
        if (k ? p.k.gamma != nullptr : p.q.gamma != nullptr) {
          const float r = rsqrtf(q / (float)p.dim + p.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] *= r * (float)(k ? ga[1][i] : ga[0][i]);
            y[i] *= r * (float)(k ? gb[1][i] : gb[0][i]);
          }
        }
      }
      f16x8 oa, ob;
      if (!turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          oa[i] = (f16)x[i];
          ob[i] = (f16)y[i];
        }
      } else if (p.interleaved) {  // pairs (x0, x1), (x2, x3), ... (y0, y1), ...
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          oa[i] = (f16)(x[i] * c[i / 2] - x[i + 1] * s[i / 2]);
          oa[i + 1] = (f16)(x[i + 1] * c[i / 2] + x[i] * s[i / 2]);
          ob[i] = (f16)(y[i] * c[4 + i / 2] - y[i + 1] * s[4 + i / 2]);
          ob[i + 1] = (f16)(y[i + 1] * c[4 + i / 2] + y[i] * s[4 + i / 2]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          oa[i] = (f16)(x[i] * c[i] - y[i] * s[i]);
          ob[i] = (f16)(y[i] * c[i] + x[i] * s[i]);
        }
      }
      if (at[e].kind < 2 && has_a) *reinterpret_cast<f16x8*>(at[e].y + ca) = oa;
      if (at[e].kind < 2 && has_b) *reinterpret_cast<f16x8*>(at[e].y + cb) = ob;
    }
  }
}

// Any sizes and alignment: a wavefront a head, an element or a pair a lane.
__global__ __launch_bounds__(64 * kWaves) void rope_any_kernel(RopeParams p, RopeSteps steps) {
  __shared__ float2 lds[kWaves][kMaxRopePairs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kWaves + wave;
  const int row = p.row0 + (int)w;
  if (row >= p.rows) return;
  int64_t out_row = row;
  if (p.kv_rows) out_row = p.kv_rows[row];
  const bool kv_on = !p.kv_rows || (out_row >= 0 && out_row < p.kv_out_rows);
  const int position = p.rot == 0 ? 0 : p.positions ? p.positions[row] : row % p.seq;
  float2* cs = lds[wave];
  angles(p, steps, position, cs, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const int pairs = p.rot / 2;
  auto heads = [&](const RopeParams::Part& t, int64_t yr, bool turn) {
    for (int h = 0; h < t.heads; ++h) {
      const f16* x = t.x + row * t.x_row + h * t.x_head;
      f16* y = t.y + yr * t.y_row + h * t.y_head;
      float pa[2] = {}, pb[2] = {}, rest[4] = {};
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
          rest[e] = (float)x[d];
          q = fmaf(rest[e], rest[e], q);
        }
      }
      const bool norm = turn && t.gamma;
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
          const float2 a = turn ? cs[i] : make_float2(1.f, 0.f);
          y[ia] = (f16)(turn ? u * a.x - v * a.y : u);
          y[ib] = (f16)(turn ? v * a.x + u * a.y : v);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = p.rot + lane + 64 * e;
        if (d < p.dim) y[d] = (f16)(norm ? rest[e] * (r * (float)t.gamma[d]) : rest[e]);
      }
    }
  };
  heads(p.q, row, true);
  if (kv_on) {
    heads(p.k, out_row, true);
    heads(p.v, out_row, false);
  }
}

bool wide(const RopeParams::Part& t) {
  if (!t.heads) return true;
  return (((uintptr_t)t.x | (uintptr_t)t.y) & 15) == 0 &&
         ((t.x_row | t.x_head | t.y_row | t.y_head) & 7) == 0;
}

template <int G>
hipError_t launch(const RopeParams& p, const RopeSteps& steps, int rows, hipStream_t s) {
  const int heads = p.q.heads + p.k.heads + p.v.heads, at_once = 64 / G;
  // few rows: their heads over several wavefronts
  const int most = (heads + at_once - 1) / at_once;
  const int waves = std::min(most, std::max(1, 4096 / rows));
  const dim3 grid((unsigned)(((int64_t)rows * waves + kWaves - 1) / kWaves)), block(64 * kWaves);
  if (p.q.gamma || p.k.gamma)
    hipLaunchKernelGGL((rope_kernel<G, true>), grid, block, 0, s, p, steps, waves);
  else
    hipLaunchKernelGGL((rope_kernel<G, false>), grid, block, 0, s, p, steps, waves);
  return hipGetLastError();
}

}  // namespace

hipError_t rope_heads(const RopeParams& args, const RopeSteps& steps, hipStream_t s) {
  const bool fast = args.dim % 8 == 0 && args.rot % 16 == 0 && wide(args.q) && wide(args.k) &&
                    wide(args.v);
  constexpr int kRows = 1 << 25;  // of a launch, whose threads are counted in 32 bits
  for (int row0 = 0; row0 < args.rows;) {
    RopeParams p = args;
    const int rows = std::min(kRows, args.rows - row0);
    p.row0 = row0;
    p.rows = row0 + rows;
    hipError_t e;
    if (!fast) {
      hipLaunchKernelGGL(rope_any_kernel, dim3((unsigned)((rows + kWaves - 1) / kWaves)),
                         dim3(64 * kWaves), 0, s, p, steps);
      e = hipGetLastError();
    } else {
      e = p.dim <= 16    ? launch<1>(p, steps, rows, s)
          : p.dim <= 32  ? launch<2>(p, steps, rows, s)
          : p.dim <= 64  ? launch<4>(p, steps, rows, s)
          : p.dim <= 128 ? launch<8>(p, steps, rows, s)
                         : launch<16>(p, steps, rows, s);
    }
    if (e != hipSuccess) return e;
    row0 += rows;
  }
  return hipSuccess;
}

}  // namespace bbh

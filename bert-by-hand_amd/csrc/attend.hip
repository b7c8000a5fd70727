// Attention for models other than MiniLM: any head size up to 256, shared
// key/value heads, capped scores, a bias by distance, a window, a prefix, a key
// mask, documents packed end to end, and few queries over a long cache.
//
// Mathematics.  One pass over the keys with a running maximum m, sum l and output o for each
// row (a query of a head), in base 2: for each tile of keys
//   s = q K^T,  w = 2^(mscale s - m),  l += sum w,  o += w V,
// where o and l are rescaled only when m rises by more than kLazy.  A cap's tanh is 1 - 2 / (1 + e^2x):
// the constant drops out of the softmax, and one exp2 and one reciprocal are left, for caps of up
// to kNearCap (shape()).
//
// Rows.  A wavefront has 32 rows: the heads that share a key/value head lie side by side in them
// (row = query * group + head), so that a tile of K and V serves all of them, and one token of 8
// heads fills 8 rows where a row a query would leave 31 empty.
//
// Layout.  Scores are computed as S^T = K Q^T (32x32x16): a lane then has 16 scores of ONE row,
// the maximum takes one exchange between lanes, and the weights are, in the lane that computed them,
// the operand of the second product O^T = V^T W^T, given that K's rows lie permuted in LDS
// (key_of_row).  V^T comes from rows of V by transposed LDS reads.  K and V go to LDS by buffer
// loads without passing registers; chunks of 16 bytes lie XORed by the row so that the reads of
// both hit all banks evenly; rows behind the last key and values behind the head's size are past the
// resource's end and become zeros.
//
// What bounds it (the cases as sequences x tokens x heads (key/value heads) x head size, fp16):
//  8192 causal, 32 (8) x 128  535-555 us, 990-1030 TFLOP/s of the 1311 that a library product of
//                             8192^3 reaches: matrix cores busy half of the time, vector units 38%
//                             (exponentials first); one wavefront's softmax runs beside another's
//                             products, at 1.65-1.7 GHz.
//  4 x 4096, window of 1023, prefix, cap, 16 (4) x 256  471 us, 543 TFLOP/s: 32 rows of 256 values
//                             leave one wavefront a SIMD, whose products and softmax take turns.
//  64 tokens over caches of up to 8192, 32 (8) x 128  187 us, 4.8 TB/s of K and V.
//  heads of 64 and short sequences: a tile's steps one after another (vector units 37-54% busy by
//                             instructions, matrix cores 10-16%) and each workgroup's start.
#include <limits.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attend.h"
#include "pipe.h"

namespace bbh {
namespace {

#define BBH_LDS __attribute__((address_space(3)))
typedef BBH_LDS f16 lds_f16;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// A softmax of the products, of ones under a cap up to kNearCap, with any bias beside them, with a
// larger cap and any bias.
enum Feat { kPlain = 0, kCap = 1, kAny = 2, kWide = 3 };

// Key (within a 32-key chunk) held by row r of the K tile.
__device__ __forceinline__ int key_of_row(int r) {
  const int a = r >> 3, c = (r >> 2) & 1, b = r & 3;
  return 16 * (a >> 1) + 8 * c + 4 * (a & 1) + b;
}

// Chunk c (16 bytes) of a row r of a tile of HD-wide rows sits in slot c ^ f(r).
template <int HD>
struct Tile {
  static constexpr int CPR = HD / 8;
  __device__ static __forceinline__ int fk(int r) {
    if constexpr (HD % 128 == 0) return r & 15;
    if constexpr (HD % 64 == 0) return (r >> 1) & 7;
    return (r >> 2) & 3;
  }
  __device__ static __forceinline__ int fv(int r) {
    if constexpr (HD % 128 == 0) return 4 * (r & 3);
    if constexpr (HD % 64 == 0) return 4 * ((r >> 1) & 1);
    return 0;
  }
};

constexpr float kLazy = 8.f;
// Weights are 2^kRoom times what they are called here, up to 2^15 with kLazy: the factor is in the
// sums and the output alike, and fp16, which weights are rounded to for the product with V, holds
// ones down to 2^-21 of a row's maximum to 2^-11 of themselves, and smaller ones to 2^-32 of that (2^-25
// without: at 10^5 equal keys e^18 below one other, all of them were zeros there and none in the sum).
constexpr float kRoom = 7.f;
// A weight's exponent is fma(mscale, s, -(m mscale rounded)): one operation, and the product's
// rounding error, the same in all of a row's weights, cancels with their sum.  With scores of 2^28
// and more that error would itself be far from 0 (a bias of the type's lowest value: 2^100).  So
// while a wavefront's maxima lie further out than kFar, they are subtracted from the scores before
// anything is scaled: exact next to the maximum.  Maxima stay what they are, never counted from an
// earlier one: a score near 0 behind one of -10^9 would lose its digits in such a difference.
constexpr float kFar = 65536.f;
constexpr int kMaxSplits = 256;  // a thread of the joining workgroup each

template <int HD_, int NW_, int KS_, int SK_, int R_, int OCC_>
struct Cfg {
  static constexpr int HD = HD_, NW = NW_, KS = KS_, R = R_, OCC = OCC_;
  static_assert(KS == 1 || KS == NW, "waves go along the rows or along the keys");
  static constexpr int RW = NW / KS;
  static constexpr int BM = RW * 32;             // rows of a workgroup
  static constexpr int SK = SK_;                 // keys of a tile
  static constexpr int CH = SK / 32;             // 32-key chunks of a tile
  static constexpr int CW = KS == 1 ? NW : 1;    // wavefronts that share a tile's copies
  static constexpr int N = SK * HD / 512 / CW;   // copies of a wavefront: a tile of K, of V
  static_assert(SK * HD % (512 * CW) == 0, "whole copies a wavefront");
  static constexpr int STAGE = 2 * SK * HD;      // halves of a stage: K, V
  static constexpr int RINGS = KS;               // a ring each wavefront where it has tiles of its own
  static constexpr size_t RING = (size_t)RINGS * R * STAGE * 2;
  static constexpr size_t OUT = KS == 1 ? (size_t)NW * 32 * (HD + 8) * 2
                                        : (size_t)KS * 32 * (HD + 4) * 4 + KS * 32 * 8;
  static constexpr size_t MASKS = (size_t)RINGS * R * 64 * 4;  // a tile's mask beside it
  static constexpr size_t LDS = RING + MASKS > OUT ? RING + MASKS : OUT;
  static constexpr int THREADS = 64 * NW;
};

struct Seq {
  int64_t q0, k0;  // first row (packed) of queries and keys
  int nq, nk;
};

// Rows of sequence b, inside the tensor whatever the offsets hold (both ends clamped: their
// difference then fits an int) and whatever the length.
__device__ __forceinline__ int span_of(const int32_t* offsets, const int32_t* lengths, int b,
                                       int len, int64_t rows, int64_t& start) {
  start = 0;
  int n = len;
  if (offsets) {
    const int64_t a = offsets[b], e = offsets[b + 1];
    start = a < 0 ? 0 : a > rows ? rows : a;
    const int64_t end = e < 0 ? 0 : e > rows ? rows : e;
    n = (int)(end - start < len ? end - start : len);
  }
  if (lengths) n = min(n, lengths[b]);
  return max(n, 0);
}
// n / d for any 32-bit n, with the host's ceil(2^64 / d) (0: d is 1): a division takes some thirty
// instructions, as many as part of a short sequence's tile.
__device__ __forceinline__ int divide(int n, Divisor d) {
  if ((d.hi | d.lo) == 0) return n;
  const uint64_t low = (uint64_t)(uint32_t)n * d.lo, high = (uint64_t)(uint32_t)n * d.hi;
  return (int)((high + (low >> 32)) >> 32);
}
// row / group: rows of up to 2^28 by groups of up to 16 with one multiplication (a division
// takes forty instructions, as many as a short sequence's tile).
__device__ __forceinline__ int query_of(const AttendParams& p, int row) {
  if (p.group == 1) return row;
  return p.group_magic ? (int)__umulhi((uint32_t)row, p.group_magic) : row / p.group;
}
__device__ __forceinline__ Seq seq_of(const AttendParams& p, int b) {
  Seq s;
  s.nq = span_of(p.q_offsets, p.q_lengths, b, p.q_len, p.q_rows, s.q0);
  s.nk = span_of(p.k_offsets, p.k_lengths, b, p.k_len, p.k_rows, s.k0);
  return s;
}

__device__ __forceinline__ int wave_id() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}
__device__ __forceinline__ float imax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

struct IeeeMax {
  __device__ __forceinline__ float operator()(float a, float b) const { return imax(a, b); }
};

// Scheduling of STEPS steps, each of READS LDS reads and a product of what they read: the reads
// run A steps ahead of the products, no further (left alone the compiler reads the whole tile
// first, into more registers than there are).  VALU and TRANS other operations of the block go
// beside each product.
template <int STEPS, int READS, int A, int VALU = 0, int TRANS = 0>
__device__ __forceinline__ void ahead() {
  constexpr int P = A < STEPS ? A : STEPS;
  __builtin_amdgcn_sched_group_barrier(0x100, READS * P, 0);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i + P < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    if constexpr (VALU > 0) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    if constexpr (TRANS > 0) __builtin_amdgcn_sched_group_barrier(0x400, TRANS, 0);
  }
}
constexpr int kAheadK = 4, kAheadV = 4;

// What a lane knows of its row (a wavefront has 32 rows; lanes l and l + 32 share one), and the
// running state of its softmax.  m is in the units that shape() leaves the scores in; times mscale
// they are powers of two.
template <class C>
struct Row {
  f16x8 q[C::HD / 16];
  int lo, hi;  // keys it sees, apart from the prefix
  int pos;
  int first, last;  // of the wavefront's rows: least and largest position
  float slope;
  int tab;  // where distance 0 of the head's table is in LDS, or the head (a table in memory)
  f32x16 o[C::HD / 32];  // o[d][i]: dim 32 d + 8 (i / 4) + 4 (lane / 32) + i % 4
  float m, l;
  float mc;   // m * mscale (0 where m is subtracted, or -infinity) - kRoom: a weight's exponent 0
  float lag;  // how far above m scores may lie: kLazy / mscale, or none at all (-infinity) while
              // some row's m lies further from 0 than kFar
};
// A bias in the units of the scores.  Finite ones stay finite, in those units and as powers of two.
__device__ __forceinline__ float bias_units(const AttendParams& p, float w) {
  return w == -INFINITY ? w : imax(imax(w, -1e38f) * p.bias_scale, -1e38f);
}
// The scores of a tile: s[ch][i] is key 32 ch + 16 (i / 8) + 8 (lane / 32) + i % 8 of it.
template <class C>
struct Scores {
  f32x16 s[C::CH];
};
template <class C>
struct Weights {
  f16x8 w[C::CH][2];
};

// Scores of the tile at LDS rows ks (K, chunked by fk).
template <class C>
__device__ __forceinline__ void scores(const Row<C>& r, const lds_f16* __restrict__ ks, Scores<C>& x) {
  const int lane = threadIdx.x & 63, r32 = lane & 31, kh = lane >> 5;
#pragma unroll
  for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
    for (int st = 0; st < C::HD / 16; ++st) {
      const f16x8 kf = *reinterpret_cast<const BBH_LDS f16x8*>(
          ks + (32 * ch + r32) * C::HD + (((2 * st + kh) ^ Tile<C::HD>::fk(r32)) << 3));
      x.s[ch] = mfma32(kf, r.q[st], st == 0 ? f32x16{} : x.s[ch]);
    }
}

// Cap and bias.  The products s of q and k become -1 / (1 + 2^(cap_k s)) under a cap, which rises
// as tanh does and times 2 cap is cap * tanh but for a constant, which a softmax does not see.
// Biases arrive in the units of either (divided by mscale), so that nothing is scaled here.
//
// That value lies near -1/2 wherever s is small against the cap, so that a score is off by up to
// 8 * 2^-24 of the cap: 6e-5 at kNearCap, an eighth of a rounding of the weights to fp16, but more
// than 1 at 2^24.  Under larger caps the value is tanh(x) itself, off by 2^-21 of its own size: up
// to 3/4 the quotient x (945 + 105 x^2 + x^4) / (945 + 420 x^2 + 15 x^4), a convergent of tanh's
// continued fraction (3e-9 of it at 3/4), from there on 1 - 2 / (1 + e^2|x|).  These are three
// times the operations, in kernels of their own: beside the others' they take registers that cost
// 5-15% of calls with a bias (4 x 4096 causal, 16 (4) x 128: 312 us without a cap, 374 up to kNearCap,
// 550 beyond).
__device__ __forceinline__ float tanh_of(float x) {
  const float a = fabsf(x), x2 = x * x;
  const float n = fmaf(x2, x2 + 105.f, 945.f), d = fmaf(x2, fmaf(x2, 15.f, 420.f), 945.f);
  const float e = __builtin_amdgcn_exp2f(a * 2.8853900817779268f);  // 2 log2(e)
  const float far = copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + e), 1.f), x);
  return a < 0.75f ? x * n * __builtin_amdgcn_rcpf(d) : far;
}

// The table of a head lies in LDS with its ends repeated kPad times, so that the distances of a
// chunk (32 keys from at most 32 neighbouring queries: 62 apart at most) are either all past one
// end, where the bias is a constant, or all inside the padded table, where a lane reads eight
// neighbouring values with no clamping.  Tables of more than 16 KB are read from memory, so that
// every set keeps its workgroups a CU (32 x 509, 12 x 64, us: 257 entries 52.7, 1801 57.0, 3801 61.6;
// from memory, 3969 to 18001, 88.9).
constexpr int kPad = 64;
template <class C>
__device__ __forceinline__ BBH_LDS float* table_area() {
  HIP_DYNAMIC_SHARED(f16, smem);
  return (BBH_LDS float*)((BBH_LDS char*)smem + C::LDS);
}
template <class C, int FEAT>
__device__ __forceinline__ void shape(const AttendParams& p, const Row<C>& r, int k0, Scores<C>& x) {
  if constexpr (FEAT == kPlain) return;
  const int kh = (threadIdx.x & 63) >> 5;
  if constexpr (FEAT == kWide) {
#pragma unroll
    for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
      for (int i = 0; i < 16; ++i) x.s[ch][i] = tanh_of(x.s[ch][i] * p.cap_k);
  } else if (FEAT == kCap || p.cap_k > 0.f) {
#pragma unroll
    for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        x.s[ch][i] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x.s[ch][i] * p.cap_k));
  }
  if constexpr (FEAT >= kAny) {
    if (p.slopes) {
#pragma unroll
      for (int ch = 0; ch < C::CH; ++ch) {
        const float df = (float)(k0 + 32 * ch + 8 * kh - r.pos);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x.s[ch][i] = fmaf(-r.slope, fabsf(df + (float)(16 * (i >> 3) + (i & 7))), x.s[ch][i]);
      }
    }
    if (p.table) {
#pragma unroll
      for (int ch = 0; ch < C::CH; ++ch) {
        const int kb = k0 + 32 * ch;
        const bool past = kb + 31 - r.first <= -p.half || kb - r.last >= p.half;
        const int end = kb < r.last ? -p.half : p.half;
        if (p.table_lds) {
          const BBH_LDS float* t = table_area<C>() + r.tab + (past ? end : kb + 8 * kh - r.pos);
          if (past) {
            const float w = *t;
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[ch][i] += w;
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[ch][i] += t[16 * (i >> 3) + (i & 7)];
          }
        } else {
          const float* t = p.table + (int64_t)r.tab * (2 * p.half + 1) + p.half;
          if (past) {
            const float w = bias_units(p, t[end]);
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[ch][i] += w;
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int d = kb + 8 * kh - r.pos + 16 * (i >> 3) + (i & 7);
              x.s[ch][i] += bias_units(p, t[min(max(d, -p.half), p.half)]);
            }
          }
        }
      }
    }
  }
}

// The pairs of a tile that are seen, as bits of the lane's scores; false: none of the wavefront's.
template <class C>
struct Seen {
  uint32_t bits[C::CH];
};
template <class C>
__device__ __forceinline__ bool seen_of(const Row<C>& r, int k0, uint64_t on, int prefix, Seen<C>& see) {
  const int kh = (threadIdx.x & 63) >> 5;
  uint32_t some = 0;
#pragma unroll
  for (int ch = 0; ch < C::CH; ++ch) {
    const int kb = k0 + 32 * ch;
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; };
    const uint32_t w = ((below(r.hi - kb) & ~below(r.lo - kb)) | below(prefix - kb)) &
                       (uint32_t)(on >> (32 * ch));
    some |= w;
    see.bits[ch] = w >> (8 * kh);
  }
  return __ballot(some != 0) != 0;
}
// -infinity over the scores of pairs that are not seen: a bit spread over the word, and a bitwise
// choice by it (two operations, none of them on a condition register).
template <class C>
__device__ __forceinline__ void hide(const Seen<C>& see, Scores<C>& x) {
#pragma unroll
  for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t on = (uint32_t)((int)(see.bits[ch] << (31 - 16 * (i >> 3) - (i & 7))) >> 31);
      x.s[ch][i] = __uint_as_float((on & __float_as_uint(x.s[ch][i])) | (~on & 0xff800000u));
    }
}

// Four chains: an operation on the one before's result waits twice as long as its issue takes.
template <class C>
__device__ __forceinline__ float largest(const Scores<C>& x) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = imax(x.s[0][e], x.s[0][4 + e]);
#pragma unroll
  for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
    for (int i = ch == 0 ? 8 : 0; i < 16; i += 8)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = imax(imax(v[e], x.s[ch][i + e]), x.s[ch][i + 4 + e]);
  const float m = imax(imax(v[0], v[1]), imax(v[2], v[3]));
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return imax(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

// Brings the running maximum up to a tile's, where that is far enough above it (r.lag), and
// subtracts it from the tile's scores where some row's is far.
template <class C>
__device__ __forceinline__ void raise(Row<C>& r, Scores<C>& x, float mx, float lag, float mscale) {
  // (one condition for both: a second one beside it takes 6% of 4 x 4096 causal of 12 heads of 64)
  if (!__ballot(!(mx <= r.m + r.lag))) return;
  const float mn = imax(r.m, mx);
  if (__ballot(r.m != -INFINITY)) {  // (at the first tile there is nothing to bring along)
    const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((r.m - mn) * mscale);
    r.l *= corr;
#pragma unroll
    for (int d = 0; d < C::HD / 32; ++d) r.o[d] *= corr;
  }
  r.m = mn;
  r.mc = (mn == -INFINITY ? 0.f : mn * mscale) - kRoom;
  r.lag = lag;
  if (__ballot(fabsf(r.mc) > kFar)) {
    r.lag = -INFINITY;
    r.mc = -kRoom;
    const float by = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
      for (int i = 0; i < 16; ++i) x.s[ch][i] -= by;
  }
}

// Weights 2^(mscale (s - m) + kRoom), rounded to fp16 (half of a step of an output's own type, and
// the matrix unit's operand) for the product with V; their sum is of the unrounded ones, in fp32.
// It is added up with plain additions: a dot product of two does not run while the matrix unit is
// busy (16 of them beside another wavefront's products 104 -> 230 cycles; additions 104 -> 129).
template <class C>
__device__ __forceinline__ void weigh(Row<C>& r, const Scores<C>& x, float mscale, Weights<C>& out) {
  float sum[4] = {};
#pragma unroll
  for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(fmaf(x.s[ch][i], mscale, -r.mc));
      sum[i & 3] += e;
      out.w[ch][i >> 3][i & 7] = (f16)e;
    }
  r.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// o += V^T w of the tile at LDS rows vs (V, chunked by fv): a transposed read hands a lane
// the four keys of its dim that it supplies to the product.
template <class C>
__device__ __forceinline__ void context(Row<C>& r, const lds_f16* __restrict__ vs, const Weights<C>& x) {
  constexpr int HD = C::HD;
  const int lane = threadIdx.x & 63, kh = lane >> 5;
#pragma unroll
  for (int ch = 0; ch < C::CH; ++ch)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) {
        const int row = 32 * ch + 16 * hf + 8 * kh + ((lane >> 2) & 3);
        const int c16 = (4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ Tile<HD>::fv((lane >> 2) & 3);
        const lds_f16* at = vs + row * HD + (c16 << 3) + 4 * (lane & 1);
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((BBH_LDS s16x4*)at);
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((BBH_LDS s16x4*)(at + 4 * HD));
        const f16x8 vf = __builtin_bit_cast(f16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        r.o[d] = mfma32(vf, x.w[ch][hf], r.o[d]);
      }
}

// One wavefront's share of a tile's copies.
template <class C>
struct Copies {
  uint32_t koff[C::N], voff[C::N];
  int cwave;
  static constexpr uint32_t kNowhere = 0x80000000u;  // past every resource: reads nothing, writes zeros

  __device__ __forceinline__ void init(const AttendParams& p, int wave, int lane) {
    cwave = C::KS == 1 ? wave : 0;
#pragma unroll
    for (int j = 0; j < C::N; ++j) {
      const int s = (cwave * C::N + j) * 64 + lane, r = s / Tile<C::HD>::CPR, slot = s % Tile<C::HD>::CPR;
      const int kc = slot ^ Tile<C::HD>::fk(r & 31), vc = slot ^ Tile<C::HD>::fv(r);
      const int kr = (r & ~31) + key_of_row(r & 31);
      koff[j] = 8 * kc < p.dim ? (uint32_t)(kr * (int)p.ks.row + 8 * kc) * 2u : kNowhere;
      voff[j] = 8 * vc < p.dim ? (uint32_t)(r * (int)p.vs.row + 8 * vc) * 2u : kNowhere;
    }
  }
  // `valid` keys' K (V) from src on into a stage; rows behind them become zeros.
  __device__ __forceinline__ void issue_k(const AttendParams& p, const f16* src, int valid, lds_f16* stage) {
    const auto r = buffer_of(src, valid > 0 ? (uint32_t)((valid - 1) * (int)p.ks.row + p.dim) * 2u : 0u);
    lds_f16* to = stage + cwave * C::N * 512;
#pragma unroll
    for (int j = 0; j < C::N; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (BBH_LDS void*)(to + j * 512), 16, (int)koff[j], 0, 0, 0);
  }
  __device__ __forceinline__ void issue_v(const AttendParams& p, const f16* src, int valid, lds_f16* stage) {
    const auto r = buffer_of(src, valid > 0 ? (uint32_t)((valid - 1) * (int)p.vs.row + p.dim) * 2u : 0u);
    lds_f16* to = stage + C::SK * C::HD + cwave * C::N * 512;
#pragma unroll
    for (int j = 0; j < C::N; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (BBH_LDS void*)(to + j * 512), 16, (int)voff[j], 0, 0, 0);
  }
  // Zeros over this wavefront's part of a stage's V where no row of the workgroup sees the key: a
  // weight of 0 times what such a key holds is not always 0.
  __device__ __forceinline__ void clear_unseen(lds_f16* stage, uint64_t bits, int lane) {
    lds_f16* vs = stage + C::SK * C::HD;
#pragma unroll
    for (int j = 0; j < C::N; ++j) {
      const int s = (cwave * C::N + j) * 64 + lane;
      if (!((bits >> (s / Tile<C::HD>::CPR)) & 1))
        *reinterpret_cast<BBH_LDS f16x8*>(vs + 8 * s) = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
};

template <class C, int FEAT>
__global__ __launch_bounds__(C::THREADS, C::OCC) void attend_kernel(AttendParams p) {
  constexpr int HD = C::HD, SK = C::SK, NS = HD / 16, ND = HD / 32;
  HIP_DYNAMIC_SHARED(f16, smem);
  // (sequence, key/value head), row block and split of this workgroup
  const int rows_all = p.batch * p.kv_heads, cols = p.blocks * p.splits;
  int item, col;
  {
    const int x = blockIdx.x % kXcds, n = blockIdx.x / kXcds;
    if (rows_all >= kXcdRows) {
      const int qd = divide(n, p.by_cols);
      item = qd * kXcds + x;
      col = n - qd * cols;
      if (item >= rows_all) return;
    } else {
      const int items = rows_all * cols, each = items / kXcds, r = items % kXcds;
      if (n >= each + (x < r ? 1 : 0)) return;
      const int i = x * each + min(x, r) + n;
      item = divide(i, p.by_cols);
      col = i - item * cols;
    }
  }
  const int over = divide(col, p.by_splits);
  const int split = col - over * p.splits, block = p.blocks - 1 - over;
  const int bi = divide(item, p.by_kv), kvh = item - bi * p.kv_heads, b = p.b0 + bi;
  const Seq sq = seq_of(p, b);
  const int nq = sq.nq, nk = sq.nk, rows = nq * p.group;
  const int row0 = block * C::BM;
  if (row0 >= rows) return;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, r32 = lane & 31, kh = lane >> 5;
  const int rw = C::KS == 1 ? wave : 0;

  // ---- the rows of this lane: row = query * group + head of the group
  const int shift = nk - nq;
  const int prefix = p.prefix ? min(max(p.prefix[b], 0), nk) : 0;
  Row<C> r;
  {
    const int row = min(row0 + rw * 32 + r32, rows - 1);
    const int i = query_of(p, row), h = kvh * p.group + row - i * p.group;
    const f16* src = p.q + (p.q_offsets ? (sq.q0 + i) * p.qs.row : b * p.qs.batch + i * p.qs.row) +
                     h * p.qs.head;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      r.q[s] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (16 * s + 8 * kh < p.dim) r.q[s] = *reinterpret_cast<const f16x8*>(src + 16 * s + 8 * kh);
    }
    r.pos = i + shift;
    r.lo = p.left < 0 ? 0 : max(r.pos - p.left, 0);
    r.hi = p.right < 0 ? nk : min(r.pos + p.right + 1, nk);
    if constexpr (FEAT >= kAny) {
      const int w0 = row0 + rw * 32;
      r.first = query_of(p, min(w0, rows - 1)) + shift;
      r.last = query_of(p, min(w0 + 31, rows - 1)) + shift;
      r.slope = p.slopes ? p.slopes[h] * p.bias_scale : 0.f;
      r.tab = h;
      if (p.table) {
        if (p.table_lds) {
          const int len = 2 * p.half + 1 + 2 * kPad;
          BBH_LDS float* t = table_area<C>();
          for (int e = tid; e < p.group * len; e += C::THREADS) {
            const int g = e / len, d = e - g * len - kPad;
            t[e] = bias_units(p, p.table[(int64_t)(kvh * p.group + g) * (2 * p.half + 1) +
                                         min(max(d, 0), 2 * p.half)]);
          }
          __syncthreads();
          r.tab = (h - kvh * p.group) * len + kPad + p.half;
        }
      }
    }
  }
  // ---- the tiles of this block: those of the prefix, then those of the window
  const int first_q = query_of(p, row0), last_q = query_of(p, min(row0 + C::BM, rows) - 1);
  const int wlo = p.left < 0 ? 0 : max(first_q + shift - p.left, 0);
  const int whi = p.right < 0 ? nk : min(max(last_q + shift + p.right + 1, 0), nk);
  const int np = (prefix + SK - 1) / SK;
  const int t0 = max(np, wlo / SK), t1 = (whi + SK - 1) / SK;
  const int tiles = np + max(t1 - t0, 0);
  // per wavefront where each has its own: tiles first, first + step, ...
  int begin = split * p.chunk, end = min(tiles, begin + p.chunk);
  if constexpr (C::KS > 1) begin += wave;
  const int count = begin >= end ? 0 : (end - begin + C::KS - 1) / C::KS;
  auto key_at = [&](int i) {
    const int n = begin + i * C::KS;
    return (n < np ? n : t0 + (n - np)) * SK;
  };
  // interior tiles, which every row of the block sees whole: [full_lo, full_hi)
  const int full_lo = p.left < 0 ? 0 : max(last_q + shift - p.left, 0);
  const int full_hi = p.right < 0 ? nk : min(max(first_q + shift + p.right + 1, 0), nk);

  const f16* kbase = p.k + (p.k_offsets ? sq.k0 * p.ks.row : b * p.ks.batch) + kvh * p.ks.head;
  const f16* vbase = p.v + (p.k_offsets ? sq.k0 * p.vs.row : b * p.vs.batch) + kvh * p.vs.head;
  const int32_t* mrow = p.mask ? p.mask + (int64_t)b * p.k_len : nullptr;
  lds_f16* ring = (lds_f16*)smem + (C::KS == 1 ? 0 : wave * C::R * C::STAGE);

  Copies<C> copies;
  copies.init(p, wave, lane);
  BBH_LDS int* masks = (BBH_LDS int*)((BBH_LDS char*)smem + C::RING) + (C::KS == 1 ? 0 : wave * C::R * 64);
  // Copies of tile i into a stage (past the last tile: of nothing).
  auto copy_k = [&](int i, int stage) {
    const int k0 = key_at(i), valid = i < count ? min(nk - k0, SK) : 0;
    copies.issue_k(p, kbase + (int64_t)k0 * (int)p.ks.row, valid, ring + stage * C::STAGE);
    if (mrow && copies.cwave == C::CW - 1)  // the tile's mask beside it; zeros behind the last key
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_of(mrow, (uint32_t)nk * 4u),
                                               (BBH_LDS void*)(masks + stage * 64), 4,
                                               i < count ? (k0 + lane) * 4 : (int)Copies<C>::kNowhere, 0, 0, 0);
  };
  auto copy_v = [&](int i, int stage) {
    const int k0 = key_at(i), valid = i < count ? min(nk - k0, SK) : 0;
    copies.issue_v(p, vbase + (int64_t)k0 * (int)p.vs.row, valid, ring + stage * C::STAGE);
  };
  constexpr uint64_t kAll = SK == 64 ? ~0ull : 0xffffffffull;
  // Keys of a tile that is in place: those there are, and of them those that some row of the
  // workgroup may see.
  auto below = [](int n) -> uint64_t { return n <= 0 ? 0 : n >= SK ? kAll : (1ull << n) - 1; };
  // (one condition that is the same for all tiles: windows and prefixes often end with a tile)
  const bool some_unseen = mrow || ((wlo | prefix) & (SK - 1)) || (whi < nk && (whi & (SK - 1)));
  auto bits_of = [&](int k0, int stage, bool& unseen) -> uint64_t {
    uint64_t bits = below(nk - k0);
    unseen = false;
    if (some_unseen) {
      const uint64_t live = bits;
      if (k0 < wlo || k0 + SK > whi) bits &= (below(whi - k0) & ~below(wlo - k0)) | below(prefix - k0);
      if (mrow) bits &= __ballot(masks[stage * 64 + lane] != 0);
      unseen = bits != live;
    }
    return bits;
  };
#pragma unroll
  for (int d = 0; d < ND; ++d) r.o[d] = f32x16{};
  r.m = -INFINITY;
  r.l = r.mc = 0.f;
  const float mscale = p.mscale;
  r.lag = p.lag;
  auto whole = [&](int k0, uint64_t bits) {
    return bits == kAll && (k0 + SK <= prefix || (k0 >= full_lo && k0 + SK <= full_hi));
  };

  Scores<C> x;
  Weights<C> w;
  Seen<C> see;
  // A tile's products, softmax and output; false where no row of the wavefront sees any of it.
  auto tile_scores = [&](int k0, uint64_t bits, const lds_f16* ks, bool& edge) {
    edge = !whole(k0, bits);
    if (!bits || (edge && !seen_of(r, k0, bits, prefix, see))) return false;
    scores(r, ks, x);
    ahead<C::CH * NS, 1, kAheadK>();
    return true;
  };
  auto tile_weights = [&](int k0, bool edge) {
    shape<C, FEAT>(p, r, k0, x);
    if (edge) hide(see, x);
    raise(r, x, largest(x), p.lag, mscale);
    weigh(r, x, mscale, w);
  };
  auto tile_output = [&](const lds_f16* vs) {
    context(r, vs, w);
    ahead<C::CH * 2 * ND, 2, kAheadV>();
  };
  auto lds_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  wait_vm<0>();  // the queries: their first use is inside the loop
  if constexpr (C::R == 1) {
    // A wavefront's own tile, one stage: K of the next tile is on its way from the end of this
    // one's scores on, V from the end of its output on.  Half the LDS of two stages is twice the
    // wavefronts, and those are what keeps the memory busy here.  (A copied mask is one copy more
    // than is counted: the waits are for more than they have to be.)
    static_assert(C::CW == 1, "tiles of its own");
    copy_k(0, 0);
    copy_v(0, 0);
    for (int it = 0; it < count; ++it) {
      wait_vm<C::N>();
      asm volatile("" ::: "memory");
      const int k0 = key_at(it);
      bool unseen;
      const uint64_t bits = bits_of(k0, 0, unseen);
      bool edge;
      const bool some = tile_scores(k0, bits, ring, edge);
      lds_done();
      copy_k(it + 1, 0);
      if (some) tile_weights(k0, edge);
      wait_vm<C::N>();
      asm volatile("" ::: "memory");
      if (unseen) {
        copies.clear_unseen(ring, bits, lane);
        lds_done();
      }
      if (some) tile_output(ring + SK * HD);
      lds_done();
      copy_v(it + 1, 0);
    }
  } else {
    // R - 1 tiles on their way, shared by the workgroup's wavefronts.
    static_assert(C::KS == 1, "a barrier a tile");
    constexpr int kTile = 2 * C::N;  // copies of a tile
    for (int i = 0; i < C::R - 1; ++i) {
      copy_k(i, i);
      copy_v(i, i);
    }
    int now = 0, next = C::R - 1;  // stages of tile it and of tile it + R - 1
    for (int it = 0; it < count; ++it) {
      wait_vm<(C::R - 2) * kTile>();
      lds_barrier();
      copy_k(it + C::R - 1, next);
      copy_v(it + C::R - 1, next);
      next = next == C::R - 1 ? 0 : next + 1;
      const int k0 = key_at(it);
      bool unseen;
      const uint64_t bits = bits_of(k0, now, unseen);
      lds_f16* ks = ring + now * C::STAGE;
      if (unseen) {  // all of V is cleared before any of it is read
        copies.clear_unseen(ks, bits, lane);
        lds_barrier();
      }
      now = now == C::R - 1 ? 0 : now + 1;
      bool edge;
      if (!tile_scores(k0, bits, ks, edge)) continue;
      tile_weights(k0, edge);
      tile_output(ks + SK * HD);
    }
  }
  f32x16 (&o)[ND] = r.o;
  const float m = r.m, l = xor32_sum(r.l);

  // ---- out
  const int cpr = p.dim / 8;
  auto out_at = [&](int row) {
    const int i = query_of(p, row), g = row - i * p.group;
    return p.out + (p.q_offsets ? (sq.q0 + i) * p.os.row : b * p.os.batch + i * p.os.row) +
           (kvh * p.group + g) * p.os.head;
  };
  auto slot_of = [&](int row) {
    return (((int64_t)item * p.q_len * p.group) + row) * p.splits + split;
  };
  wait_vm<0>();
  __syncthreads();  // the rings are free
  if constexpr (C::KS == 1) {
    if (p.splits > 1) {
      const int row = row0 + rw * 32 + r32;
      if (row >= rows) return;
      const int64_t sl = slot_of(row);
      if (kh == 0) p.part_ml[sl] = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(p.part_o + sl * HD + 32 * d + 8 * j + 4 * kh) =
              f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
      return;
    }
    f16* st = smem + wave * 32 * (HD + 8);
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f16x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (f16)(o[d][4 * j + e] * inv);
        *reinterpret_cast<f16x4*>(st + r32 * (HD + 8) + 32 * d + 8 * j + 4 * kh) = w;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    for (int x = lane; x < 32 * Tile<HD>::CPR; x += 64) {
      const int rr = x / Tile<HD>::CPR, cc = x % Tile<HD>::CPR, row = row0 + rw * 32 + rr;
      const f16x8 w = *reinterpret_cast<const f16x8*>(st + rr * (HD + 8) + 8 * cc);
      if (row < rows && cc < cpr) *reinterpret_cast<f16x8*>(out_at(row) + 8 * cc) = w;
    }
  } else {
    float* area = reinterpret_cast<float*>(smem);  // [KS][32][HD + 4]
    float2* ml = reinterpret_cast<float2*>(area + C::KS * 32 * (HD + 4));
    if (kh == 0) ml[wave * 32 + r32] = make_float2(m, l);
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < C::KS; ++w) top = imax(top, ml[w * 32 + r32].x);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * mscale);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(area + (wave * 32 + r32) * (HD + 4) + 32 * d + 8 * j + 4 * kh) =
            f32x4{o[d][4 * j] * f, o[d][4 * j + 1] * f, o[d][4 * j + 2] * f, o[d][4 * j + 3] * f};
    __syncthreads();
    for (int x = tid; x < 32 * (HD / 8); x += C::THREADS) {
      const int rr = x / (HD / 8), cc = x % (HD / 8), row = row0 + rr;
      if (row >= rows || cc >= cpr) continue;
      float tp = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < C::KS; ++w) tp = imax(tp, ml[w * 32 + rr].x);
#pragma unroll
      for (int w = 0; w < C::KS; ++w) {
        const float2 a = ml[w * 32 + rr];
        sum += a.x == -INFINITY ? 0.f : a.y * __builtin_amdgcn_exp2f((a.x - tp) * mscale);
      }
      float v[8] = {};
#pragma unroll
      for (int w = 0; w < C::KS; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += area[(w * 32 + rr) * (HD + 4) + 8 * cc + e];
      if (p.splits > 1) {
        const int64_t sl = slot_of(row);
        if (cc == 0) p.part_ml[sl] = make_float2(tp, sum);
        *reinterpret_cast<f32x4*>(p.part_o + sl * HD + 8 * cc) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(p.part_o + sl * HD + 8 * cc + 4) = f32x4{v[4], v[5], v[6], v[7]};
      } else {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        f16x8 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = (f16)(v[e] * inv);
        *reinterpret_cast<f16x8*>(out_at(row) + 8 * cc) = w;
      }
    }
  }
}

// Joins the splits of a row: out = sum_s f_s o_s / sum_s f_s l_s, f_s = 2^(mscale (m_s - m)).  A
// workgroup a row: its threads weigh the splits first, all at once, then groups of HD / 8
// threads add every (256 / group)th split's outputs, and their sums are added through LDS.
// (One thread for a piece of a row, split after split: 131 us for 184 splits.)
template <int HD>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p) {
  constexpr int L = HD / 8, GR = 256 / L;
  __shared__ float w[kMaxSplits];
  __shared__ float red[2][4];
  __shared__ f32x4 sums[GR][L][2];
  const int tid = threadIdx.x, per = p.q_len * p.group;
  const int64_t slot = blockIdx.x, item = slot / per;
  const int row = (int)(slot - item * per);
  const int b = (int)(item / p.kv_heads), kvh = (int)(item - (int64_t)b * p.kv_heads);  // b0 is 0 here
  const Seq sq = seq_of(p, b);
  if (row >= sq.nq * p.group) return;
  const float2 mine = tid < p.splits ? p.part_ml[slot * p.splits + tid] : make_float2(-INFINITY, 0.f);
  const float wm = wave_reduce(mine.x, IeeeMax{});
  if ((tid & 63) == 0) red[0][tid >> 6] = wm;
  __syncthreads();
  const float top = imax(imax(red[0][0], red[0][1]), imax(red[0][2], red[0][3]));
  const float f = mine.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mine.x - top) * p.mscale);
  const float ws = wave_sum(f * mine.y);
  if ((tid & 63) == 0) red[1][tid >> 6] = ws;
  if (tid < p.splits) w[tid] = f;
  __syncthreads();
  const float sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int g = tid / L, c = tid % L;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
  if (g < GR) {
#pragma unroll 2
    for (int s = g; s < p.splits; s += GR) {
      const float ws2 = w[s];
      if (ws2 == 0.f) continue;  // an empty split, or one far below the others
      const f32x4* src = reinterpret_cast<const f32x4*>(p.part_o + (slot * p.splits + s) * HD + 8 * c);
      const f32x4 u = src[0], v = src[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = fmaf(u[e], ws2, x[e]);
        y[e] = fmaf(v[e], ws2, y[e]);
      }
    }
    sums[g][c][0] = x;
    sums[g][c][1] = y;
  }
  __syncthreads();
  if (tid >= L || 8 * tid >= p.dim) return;
  x = sums[0][tid][0];
  y = sums[0][tid][1];
#pragma unroll 4
  for (int i = 1; i < GR; ++i) {
    x += sums[i][tid][0];
    y += sums[i][tid][1];
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const int i = query_of(p, row), gh = row - i * p.group;
  f16* dst = p.out + (p.q_offsets ? (sq.q0 + i) * p.os.row : b * p.os.batch + i * p.os.row) +
             (kvh * p.group + gh) * p.os.head + 8 * tid;
  f16x8 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[e] = (f16)(x[e] * inv);
    o[4 + e] = (f16)(y[e] * inv);
  }
  *reinterpret_cast<f16x8*>(dst) = o;
}

// LDS of the padded tables of a group's heads.
int64_t table_bytes(const AttendParams& p) {
  return (int64_t)p.group * (2 * (int64_t)p.half + 1 + 2 * kPad) * 4;
}

template <class C, int FEAT>
hipError_t launch_as(const AttendParams& p, int64_t grid, hipStream_t s) {
  static std::atomic<uint64_t> set{0};  // a bit a device
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(set.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(attend_kernel<C, FEAT>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLdsMax);
    if (e != hipSuccess) return e;
    set.fetch_or(bit, std::memory_order_relaxed);
  }
  const size_t lds = C::LDS + (FEAT >= kAny && p.table_lds ? table_bytes(p) : 0);
  hipLaunchKernelGGL((attend_kernel<C, FEAT>), dim3((unsigned)grid), dim3(C::THREADS), lds, s, p);
  return hipGetLastError();
}

constexpr int64_t kMostThreads = 0xffffffffll;  // of a launch

// Longest run of keys that a sequence's rows may see: its last query stands at its last key, so that
// there are none behind the window of the first, whatever `right`, but those up to there.
int64_t longest(const AttendParams& p) {
  if (p.prefix || p.left < 0) return p.k_len;
  return std::min<int64_t>(p.k_len, (int64_t)p.left + p.q_len);
}

// Row blocks, and how a block's keys are split over workgroups where those are few.
//  - Sets whose wavefronts take tiles in turn (K), the smallest of
//    sqrt(tiles) parts: then a part's chain of tiles and the join's reading of all parts take about
//      as long (128 values, 8 pairs of a sequence and a key/value head, us by parts: 8192 keys 8 16.7,
//      16 14.4, 64 15.8; 32768 keys 8 36.7, 32 29.4, 128 34.1; 131072 keys 16 122, 64 101, 256 111);
//    four rounds of the chip's places for workgroups (1, 2 and 3 a CU, by head size);
//    what the scratch holds;
//    an odd number: the first parts, which short sequences have too, would go to the same eighth,
//      quarter or half of the chip (512 ragged pairs of up to 8192 keys: 1 part 212, 2 217, 3 192, 4
//      231, 6 194, 8 209; all of 8192: 356, 374, 373, 377, 383, 386).
//    Few keys are not worth a join: up to 1024 (512 of more than 128 values, whose tile takes
//    nearly three times as long), twice that from 49 pairs on (32 pairs over 2048 keys: 1 part 18.0,
//    3 14.8; 96: 19.2, 24.4 in 4; 192 over 1024: 19.0, 24.6 in 3; 256 values, 48 over 2048: 38.1, 26.0
//    in 4).
//  - The others: 1024 workgroups, of 512 keys each at least.
template <class C>
void plan(AttendParams& p, size_t scratch_bytes) {
  const int64_t rows = (int64_t)p.q_len * p.group, items = (int64_t)p.batch * p.kv_heads;
  p.blocks = (int)((rows + C::BM - 1) / C::BM);
  const int64_t keys = longest(p), tiles = (keys + C::SK - 1) / C::SK + 2;
  p.splits = 1;
  p.chunk = INT_MAX / 2;
  const int64_t groups = items * p.blocks;
  int64_t want, target = 1024;
  if (C::KS > 1) {
    target = 1024 * (C::HD > 128 ? 1 : C::HD > 64 ? 2 : 3);
    if (keys <= (C::HD > 128 ? 512 : 1024) * (groups > 48 ? 2 : 1)) return;
    want = (int64_t)std::sqrt((double)tiles);
  } else {
    want = tiles / (512 / C::SK);
  }
  if (groups >= target) return;
  want = std::min<int64_t>(want, (target + groups - 1) / groups);
  const int64_t a_split = items * rows * (C::HD * 4 + 8);
  want = std::min<int64_t>(std::min<int64_t>(want, kMaxSplits), (int64_t)(scratch_bytes / a_split));
  if (C::KS > 1 && want % 2 == 0) --want;
  if (want < 2) return;
  p.chunk = (int)((tiles + want - 1) / want);
  p.splits = (int)want;
}

Divisor divisor(uint64_t d) {
  if (d == 1) return {0, 0};
  const uint64_t m = ~0ull / d + 1;
  return {(uint32_t)(m >> 32), (uint32_t)m};
}

template <class C>
hipError_t launch(AttendParams p, void* scratch, size_t scratch_bytes, hipStream_t s) {
  plan<C>(p, scratch ? scratch_bytes : 0);
  const int64_t cols = (int64_t)p.blocks * p.splits;
  const int64_t slots = (int64_t)p.batch * p.kv_heads * p.q_len * p.group;
  p.part_o = static_cast<float*>(scratch);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * p.splits * C::HD);
  p.lag = kLazy / p.mscale;
  p.by_cols = divisor((uint64_t)cols);
  p.by_splits = divisor((uint64_t)p.splits);
  p.by_kv = divisor((uint64_t)p.kv_heads);
  // exact for rows below 2^32 / group
  p.group_magic = p.group > 1 && p.group <= 16 ? (uint32_t)(((1ull << 32) + p.group - 1) / p.group) : 0;
  p.table_lds = p.table && table_bytes(p) <= std::min<int64_t>(16384, (int64_t)kLdsMax - (int64_t)C::LDS);
  const int feat = p.wide_cap ? kWide : p.slopes || p.table ? kAny : p.cap_k > 0.f ? kCap : kPlain;
  // sequences a launch: its work-items are counted in 32 bits
  const int64_t per = cols * p.kv_heads * C::THREADS;
  const int most = (int)std::min<int64_t>(p.batch, std::max<int64_t>(1, (kMostThreads / per) - 8));
  const int batch = p.batch;
  for (int64_t b0 = 0; b0 < batch; b0 += most) {
    p.b0 = (int)b0;
    p.batch = std::min(most, batch - p.b0);
    const int64_t rows = (int64_t)p.batch * p.kv_heads;
    const int64_t grid = rows >= kXcdRows ? (rows + kXcds - 1) / kXcds * cols * kXcds
                                          : (rows * cols + kXcds - 1) / kXcds * kXcds;
    const hipError_t e = feat == kPlain ? launch_as<C, kPlain>(p, grid, s)
                         : feat == kCap ? launch_as<C, kCap>(p, grid, s)
                         : feat == kAny ? launch_as<C, kAny>(p, grid, s)
                                        : launch_as<C, kWide>(p, grid, s);
    if (e != hipSuccess) return e;
  }
  if (p.splits > 1) {
    p.b0 = 0;
    p.batch = batch;
    hipLaunchKernelGGL((attend_join_kernel<C::HD>), dim3((unsigned)slots), dim3(256), 0, s, p);
    return hipGetLastError();
  }
  return hipSuccess;
}

// The sets of configurations, by head size (sizes between them are padded with zeros in LDS and
// registers, never in memory):
//  P  many rows a sequence: 128 rows a workgroup, 256 for 128 values a head
//  S  fewer: 64, whose copies wait for less company
//  T  up to 16 rows: a wavefront, one stage
//  K  up to 32 rows over many keys, whose four wavefronts take tiles of keys in turn
// OCC wavefronts a SIMD, where that is worth more than the few registers that some then spill:
// 2000 documents of 12 heads of 64 with slopes 163 us at four, 177 at three; 64 sequences of 256 to
// 512 tokens, 12 heads of 96, 82 at three, 86 at two.
//               HD  NW KS SK R OCC
using P32 = Cfg<32, 4, 1, 64, 2, 4>;
using P64 = Cfg<64, 4, 1, 32, 2, 4>;
using P96 = Cfg<96, 4, 1, 64, 2, 3>;
using P128 = Cfg<128, 8, 1, 64, 2, 2>;
using P256 = Cfg<256, 4, 1, 64, 2, 1>;
using S32 = Cfg<32, 2, 1, 32, 2, 4>;
using S64 = Cfg<64, 2, 1, 32, 2, 4>;
using S96 = Cfg<96, 2, 1, 32, 2, 3>;
using S128 = Cfg<128, 2, 1, 32, 2, 2>;
using S256 = Cfg<256, 2, 1, 32, 2, 1>;
using T32 = Cfg<32, 1, 1, 32, 1, 4>;
using T64 = Cfg<64, 1, 1, 32, 1, 4>;
using T96 = Cfg<96, 1, 1, 32, 1, 3>;
using T128 = Cfg<128, 1, 1, 32, 1, 2>;
using T256 = Cfg<256, 1, 1, 32, 1, 1>;
using K32 = Cfg<32, 4, 4, 32, 1, 2>;
using K64 = Cfg<64, 4, 4, 32, 1, 2>;
using K96 = Cfg<96, 4, 4, 32, 1, 2>;
using K128 = Cfg<128, 4, 4, 32, 1, 2>;
using K256 = Cfg<256, 4, 4, 32, 1, 1>;

// By rows a sequence (on average, where documents are packed) and keys.  Measured on 40000 tokens
// of 12 heads in sequences of one length, us on P / S / T:
//   64 values a head:   8 tokens 221 / 127 / 73, 16: 118 / 70 / 49, 32: 66 / 52 / 56, 64: 52 / 54 / 59,
//                       200: 68 / 74 / 95, 500: 102 / 111 / 146
//   128 values a head:  8 tokens 1142 / 243 / 148, 16: 601 / 139 / 98, 32: 336 / 99 / 99, 128: 145 / 109 / 134,
//                       300: 210 / 156 / 209, 300 by 4 heads a key/value head: 138 / 133 / 160, 500 so: 180 / 188 / 222
template <class F>
auto with_config(const AttendParams& p, F&& f) {
  const int64_t rows = (int64_t)p.q_len * p.group, keys = longest(p);
  const int64_t items = (int64_t)p.batch * p.kv_heads;
  // (a packed tensor may have more rows than the sequences, up to any int64)
  const int64_t mean = p.q_offsets ? std::min(p.q_rows, p.batch * (int64_t)p.q_len) * p.group / p.batch : rows;
#define BBH_BY_SIZE(SET)                    \
  do {                                      \
    if (p.dim <= 32) return f(SET##32{});   \
    if (p.dim <= 64) return f(SET##64{});   \
    if (p.dim <= 96) return f(SET##96{});   \
    if (p.dim <= 128) return f(SET##128{}); \
    return f(SET##256{});                   \
  } while (0)
  // K for few rows over more than 128 keys.  But heads of more than 128 values, of which a CU holds one
  // workgroup of K, run on T, a tile at a time, where there are wavefronts enough for that and few keys
  // (8 heads a key/value head of 256, us on K / T: 520 pairs over 200 keys 36 / 26, 400: 61 / 49, 1000:
  // 115 / 108; 2100: 118 / 98, 187 / 172, 374 / 405).
  if (rows <= 32 && keys > 128 && !(p.dim > 128 && items >= 512 && keys <= 512)) BBH_BY_SIZE(K);
  if (rows <= 32 && keys > 128) BBH_BY_SIZE(T);
  if (mean <= 16) BBH_BY_SIZE(T);
  // Rows of S at most.  Sequences of one length run as fast or faster on P from about 200 rows of 64
  // values on (above), ones of 80 to 160 tokens far slower, whose last rows fill little of a
  // workgroup (300 of them, 12 heads, us on P / S: 32 values 50 / 35, 64 61 / 45, 96 87 / 58; 64 of
  // 256 to 512: 45 / 45, 63 / 63, 82 / 83).
  const int64_t most = p.dim <= 96 ? 256 : p.dim <= 128 ? 1024 : 64;
  // Above 128 values a workgroup of P has its CU to itself, so that nothing runs beside its first
  // copies and last stores: worth it over many keys only (16 heads of 256, us on P / S: 500 of 192
  // tokens 965 / 659, 100 of 203 on 4 key/value heads 244 / 222, 16 of 512 121 / 118, 30 of 1000 490 / 513).
  if (mean <= most || (p.dim > 128 && keys <= 256)) BBH_BY_SIZE(S);
  BBH_BY_SIZE(P);
#undef BBH_BY_SIZE
}

}  // namespace

hipError_t attend(AttendParams p, void* scratch, size_t scratch_bytes, hipStream_t s) {
  return with_config(p, [&](auto c) { return launch<decltype(c)>(p, scratch, scratch_bytes, s); });
}

size_t attend_scratch(const AttendParams& p) {
  return with_config(p, [&](auto c) -> size_t {
    AttendParams a = p;
    plan<decltype(c)>(a, SIZE_MAX / 2);
    if (a.splits < 2) return 0;
    return (size_t)p.batch * p.kv_heads * p.q_len * p.group * a.splits * (decltype(c)::HD * 4 + 8);
  });
}

}  // namespace bbh

// The Linear on 8-bit integers: C(M,N) = sa[m] sb[n] sum_k A[m,k] B[n,k]
// [+ bias] [GELU], both operands K-contiguous.
//
// The products are summed in int32, exactly, so any split of K or order of the
// sums gives the same integer, and with the one fp32 expression of finish()
// every kernel here gives the same bits.
//
// Matrix-core instruction: v_mfma_i32_32x32x32_i8 (twice the operations of the
// fp16 form a cycle on the same bytes).  As in gemm.hip the kernels compute the
// transposed tile D(n, m) = B . A^T, so that a lane holds runs of four
// consecutive output columns of one row.
//
// K goes in slices of 128 bytes: a row of a slice is one cache line, eight
// 16-byte chunks, and logical chunk c of row r sits in slot c ^ ((r >> 1) & 7)
// (the layout of pipe.h's 64-wide fp16 slice, byte for byte).

#include <atomic>

#include "int8.h"
#include "pipe.h"

namespace bbh {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef i32x4 i32x4_any __attribute__((aligned(1)));
typedef f16x8 f16x8_any __attribute__((aligned(2)));

constexpr int kSlice = 128;  // bytes of K a slice
constexpr int kChunk = 16;

struct Args {
  const int8_t *A, *B;
  const float *sa, *sb;
  const f16* bias;
  f16* C;
  int M, N, K;
};

// The output of one sum, the same fp32 operations wherever it is computed:
// (float) acc rounds sums of 2^24 and more, then a product and an fma.
template <bool GELU>
__device__ __forceinline__ f16 finish(int acc, float sa, float sb, float bias) {
  const float v = fmaf((float)acc * sa, sb, bias);
  return to_half(GELU ? gelu_poly(v) : v);
}

__device__ __forceinline__ int64_t block_id() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

// Workgroup -> tile of a tm x tn grid of tiles.  Each XCD gets one contiguous
// span of the tiles (workgroup b runs on XCD b % 8), in bands of kBand tile
// rows walked column by column: the 32 workgroups an XCD runs at a time then
// form a kBand x 4 block that shares kBand + 4 operand panels in its L2, where
// a row of tiles would need 33.
constexpr int kBand = 8;
__device__ __forceinline__ bool tile_of(int tm, int tn, int& bm, int& bn) {
  const int64_t b = block_id();
  const int items = tm * tn, x = (int)(b % kXcds), k = (int)(b / kXcds);
  const int q = items / kXcds, r = items % kXcds;
  if (k >= q + (x < r ? 1 : 0)) return false;
  const int item = x * q + min(x, r) + k;
  const int band = item / (kBand * tn), in = item - band * kBand * tn;
  const int rows = min(kBand, tm - band * kBand);
  bn = in / rows;
  bm = band * kBand + in - bn * rows;
  return true;
}

// A BM x BN tile by KS groups of WM x WN wavefronts; group g takes the K slices
// g, g + KS, ..., each through a ring of R slices of its own, and the groups'
// sums are added through LDS.
template <int BM_, int BN_, int WM_, int WN_, int KS_, int R_>
struct Cfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KS = KS_, R = R_;
  static constexpr int GW = WM * WN, THREADS = 64 * GW * KS;  // wavefronts a group
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  static constexpr int LA = BM / 8 / GW, LB = BN / 8 / GW, L = LA + LB;  // 1 KB copies a wavefront
  static constexpr int STAGE = (BM + BN) * kSlice;
  static constexpr int RING = STAGE * R * KS;
  static constexpr int OUT_LD = BN + 8;  // padded row of the fp16 tile (KS == 1)
  static constexpr int SUM_LD = BN + 4;  // of the groups' int32 tiles
  static constexpr int OUT = KS == 1 ? BM * OUT_LD * 2 : KS * BM * SUM_LD * 4;
  static constexpr int VEC = RING > OUT ? RING : OUT;       // sa, sb, bias follow
  static constexpr int LDS = VEC + (BM + 2 * BN) * 4;
  static constexpr int CH = (BM + BN) * 8 / (64 * GW);      // chunks a thread (unaligned)
  static_assert(TM % 32 == 0 && TN % 32 == 0, "whole 32x32 blocks");
  static_assert(BM % (8 * GW) == 0 && BN % (8 * GW) == 0, "copies");
  static_assert(R >= 2 && (R - 2) * L < 64, "vmcnt range");
  static_assert(LDS <= (int)kLdsMax && THREADS <= 1024, "workgroup");
};

// Copies of this wavefront's share of a slice: global -> LDS, 1 KB = 8 rows a
// copy.  Rows and bytes past the operand are out of the resource's bounds, as
// is everything at an offset of kNowhere: such copies read no memory.
constexpr uint32_t kNowhere = 1u << 30;
struct Copier {
  __amdgpu_buffer_rsrc_t src;
  uint32_t lane[2], step;  // byte offset in an even / odd block of 8 rows; 8 rows
  __device__ __forceinline__ Copier(const int8_t* base, int rows, int K)
      : src(buffer_of(base, (uint32_t)rows * K)), step(8u * K) {
    const int l = threadIdx.x & 63, r = l >> 3;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      lane[p] = r * K + (((l & 7) ^ (p << 2 | r >> 1)) << 4);
  }
  template <int N>
  __device__ __forceinline__ void copy(uint32_t at, char* dst, int wave) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int b = wave * N + j;  // block of 8 rows
      const uint32_t off = (N % 2 == 0 ? lane[j & 1] : lane[b & 1]) + (b * step + at);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          src, (__attribute__((address_space(3))) void*)(dst + b * 1024), 16, (int)off, 0, 0, 0);
    }
  }
};

template <class C>
struct Frags {
  i32x4 a[C::FM], b[C::FN];
  // K step j (32 bytes) of the slice at `st`; lane l reads row l % 32, chunk
  // 2 j + l / 32.
  __device__ __forceinline__ void read(const char* st, int j, int at, int wm, int wn) {
    const char* p = st + (at ^ (j << 5));
#pragma unroll
    for (int f = 0; f < C::FM; ++f)
      a[f] = *reinterpret_cast<const i32x4*>(p + (wm * C::TM + f * 32) * kSlice);
#pragma unroll
    for (int f = 0; f < C::FN; ++f)
      b[f] = *reinterpret_cast<const i32x4*>(p + (C::BM + wn * C::TN + f * 32) * kSlice);
  }
  __device__ __forceinline__ void mul(i32x16 (&acc)[C::FM][C::FN]) const {
#pragma unroll
    for (int fm = 0; fm < C::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < C::FN; ++fn)
        acc[fm][fn] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[fn], a[fm], acc[fm][fn], 0, 0, 0);
  }
};

// Scheduling groups: (one LDS read, then ~Q / R matrix products) x R.
template <int R, int Q, int I = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (I < R) {
    constexpr int n = (I < Q % R) ? Q / R + 1 : Q / R;
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x008, n, 0);
    interleave<R, Q, I + 1>();
  }
}

// 16 bytes at k of a row of K, zeros past its end.
__device__ __forceinline__ i32x4 load_chunk(const int8_t* row, int k, int K) {
  i32x4 v = {0, 0, 0, 0};
  if (k + kChunk <= K) {
    v = *reinterpret_cast<const i32x4_any*>(row + k);
  } else if (k < K) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 15; ++e)
      if (k + e < K) w[e / 4] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e % 4));
    v = i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
  }
  return v;
}

// ALIGNED: K % 16 == 0 and 16-byte aligned operands; the slices are copied
// global -> LDS with buffer loads to LDS.  Otherwise they go through registers,
// one slice ahead, the bytes past K cleared.
template <class C, bool ALIGNED, bool GELU>
__global__ __launch_bounds__(C::THREADS) void gemm_i8_kernel(Args g, int tm, int tn) {
  extern __shared__ __align__(16) char smem[];
  int bm, bn;
  if (!tile_of(tm, tn, bm, bn)) return;
  const int K = g.K, m0 = bm * C::BM, n0 = bn * C::BN;
  const int rows = min(C::BM, g.M - m0), cols = min(C::BN, g.N - n0);
  const int8_t* A = g.A + (size_t)m0 * K;
  const int8_t* B = g.B + (size_t)n0 * K;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int grp = wave / C::GW, w = wave % C::GW, wm = w / C::WN, wn = w % C::WN;

  float* vsa = reinterpret_cast<float*>(smem + C::VEC);
  float* vsb = vsa + C::BM;
  float* vbias = vsb + C::BN;
  for (int i = threadIdx.x; i < C::BM; i += C::THREADS) vsa[i] = i < rows ? g.sa[m0 + i] : 0.f;
  for (int i = threadIdx.x; i < C::BN; i += C::THREADS) {
    vsb[i] = i < cols ? g.sb[n0 + i] : 0.f;
    vbias[i] = i < cols && g.bias ? (float)g.bias[n0 + i] : 0.f;
  }

  i32x16 acc[C::FM][C::FN];
#pragma unroll
  for (int fm = 0; fm < C::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < C::FN; ++fn)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[fm][fn][i] = 0;

  // Iteration i of a group is slice i * KS + grp.  Every group has `even` whole
  // slices; then one iteration more, in which a group has a whole slice, the
  // last part of K or none, unless no group has any.
  const int full = K / kSlice, rem = K % kSlice, total = full + (rem ? 1 : 0);
  const int even = full / C::KS, iters = (total + C::KS - 1) / C::KS;
  char* const ring = smem + grp * C::R * C::STAGE;
  char* const ring_end = ring + C::R * C::STAGE;
  const Copier ca(A, rows, K), cb(B, cols, K);
  auto issue = [&](int i, char* dst) {  // ALIGNED: the slice of iteration i into a slot
    const int s = i * C::KS + grp;
    const uint32_t at = s < total ? (uint32_t)s * kSlice : kNowhere;
    ca.template copy<C::LA>(at, dst, w);
    cb.template copy<C::LB>(at, dst + C::BM * kSlice, w);
  };
  i32x4 held[ALIGNED ? 1 : C::CH];
  auto load = [&](int i) {  // the same into registers
    const int s = i * C::KS + grp;
#pragma unroll
    for (int j = 0; j < C::CH; ++j) {
      const int q = w * 64 + lane + j * 64 * C::GW, r = q >> 3, k = s * kSlice + (q & 7) * kChunk;
      // rows past the tile's last: that one again (nothing of theirs is written)
      const int8_t* row = r < C::BM ? A + (size_t)min(r, rows - 1) * K
                                    : B + (size_t)min(r - C::BM, cols - 1) * K;
      if (s < full)
        held[j] = *reinterpret_cast<const i32x4_any*>(row + k);
      else
        held[j] = load_chunk(row, k, K);
    }
  };
  auto put = [&](char* dst) {
#pragma unroll
    for (int j = 0; j < C::CH; ++j) {
      const int q = w * 64 + lane + j * 64 * C::GW, r = q >> 3;
      *reinterpret_cast<i32x4*>(dst + r * kSlice + (((q & 7) ^ (r >> 1 & 7)) << 4)) = held[j];
    }
  };
  auto next = [&](char* p) { return p + C::STAGE == ring_end ? ring : p + C::STAGE; };
  char* slot = ring;      // of the slice that is read
  char* refill = ring;    // the slot that the next copies go to
  if constexpr (ALIGNED) {
#pragma unroll
    for (int i = 0; i < C::R - 1; ++i) issue(i, ring + i * C::STAGE);
    refill = ring_end - C::STAGE;
  } else {
    load(0);
  }

  const int r32 = lane & 31, at = r32 * kSlice + ((lane >> 5 ^ (r32 >> 1 & 7)) << 4);
  // Makes slice i readable: its copies have landed (those of the R - 2 later
  // ones may be in flight), and every wavefront has read slice i - 1, whose
  // slot the next copies fill.
  auto arrive = [&](int) {
    if constexpr (ALIGNED)
      wait_vm<(C::R - 2) * C::L>();
    else
      put(slot);
    lds_barrier();
  };
  auto advance = [&](int i) {  // the copies that follow arrive(i)
    if constexpr (ALIGNED) {
      issue(i + C::R - 1, refill);
      refill = next(refill);
    } else if (i + 1 < iters) {
      load(i + 1);
    }
  };
  Frags<C> f0, f1;
  constexpr int RD = C::FM + C::FN, MF = C::FM * C::FN;
  // K steps 0-2 of the slice, each beside the reads of the next step.
  auto three = [&] {
    __builtin_amdgcn_sched_barrier(0);
    f1.read(slot, 1, at, wm, wn);
    f0.mul(acc);
    interleave<RD, MF>();
    __builtin_amdgcn_sched_barrier(0);
    f0.read(slot, 2, at, wm, wn);
    f1.mul(acc);
    interleave<RD, MF>();
    __builtin_amdgcn_sched_barrier(0);
    f1.read(slot, 3, at, wm, wn);
    f0.mul(acc);
    interleave<RD, MF>();
    __builtin_amdgcn_sched_barrier(0);
    slot = next(slot);
  };
  if (even > 0) {
    arrive(0);
    f0.read(slot, 0, at, wm, wn);
    advance(0);
    for (int i = 1; i < even; ++i) {
      three();
      arrive(i);
      f0.read(slot, 0, at, wm, wn);
      advance(i);
      f1.mul(acc);
      interleave<RD, MF>();
    }
    three();
    f1.mul(acc);
  }
  if (iters > even) {
    arrive(even);
    const int s = even * C::KS + grp, left = min(kSlice, K - s * kSlice);
    for (int j = 0; j * 32 < left; ++j) {
      f0.read(slot, j, at, wm, wn);
      // past K: the next row's bytes in both operands, cleared in one
      if (ALIGNED && (2 * j + (lane >> 5)) * kChunk >= left)
#pragma unroll
        for (int f = 0; f < C::FM; ++f) f0.a[f] = i32x4{0, 0, 0, 0};
      f0.mul(acc);
    }
  }
  if constexpr (ALIGNED) wait_vm<0>();  // copies from nowhere are still copies
  lds_barrier();                        // the ring is free

  if constexpr (C::KS == 1) {
    f16* out = reinterpret_cast<f16*>(smem);
#pragma unroll
    for (int fm = 0; fm < C::FM; ++fm) {
      const int m = wm * C::TM + fm * 32 + r32;
      const float sa = vsa[m];
#pragma unroll
      for (int fn = 0; fn < C::FN; ++fn)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = wn * C::TN + fn * 32 + 8 * q + 4 * (lane >> 5);
          const f32x4 sb = *reinterpret_cast<const f32x4*>(vsb + n);
          const f32x4 bi = *reinterpret_cast<const f32x4*>(vbias + n);
          f16x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = finish<GELU>(acc[fm][fn][4 * q + e], sa, sb[e], bi[e]);
          *reinterpret_cast<f16x4*>(out + m * C::OUT_LD + n) = o;
        }
    }
  } else {
    int* sums = reinterpret_cast<int*>(smem) + grp * C::BM * C::SUM_LD;
#pragma unroll
    for (int fm = 0; fm < C::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < C::FN; ++fn)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = wm * C::TM + fm * 32 + r32;
          const int n = wn * C::TN + fn * 32 + 8 * q + 4 * (lane >> 5);
          *reinterpret_cast<i32x4*>(sums + m * C::SUM_LD + n) =
              i32x4{acc[fm][fn][4 * q], acc[fm][fn][4 * q + 1], acc[fm][fn][4 * q + 2],
                    acc[fm][fn][4 * q + 3]};
        }
  }
  lds_barrier();
  for (int i = threadIdx.x; i < C::BM * C::BN / 8; i += C::THREADS) {
    const int m = i / (C::BN / 8), n = i % (C::BN / 8) * 8;
    if (m >= rows || n >= cols) continue;
    f16x8 o;
    if constexpr (C::KS == 1) {
      o = *reinterpret_cast<const f16x8*>(reinterpret_cast<const f16*>(smem) + m * C::OUT_LD + n);
    } else {
      int v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < C::KS; ++k) {
        const int* p = reinterpret_cast<const int*>(smem) + (k * C::BM + m) * C::SUM_LD + n;
        const i32x4 x = *reinterpret_cast<const i32x4*>(p), y = *reinterpret_cast<const i32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += x[e];
          v[4 + e] += y[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = finish<GELU>(v[e], vsa[m], vsb[n + e], vbias[n + e]);
    }
    f16* dst = g.C + (size_t)(m0 + m) * g.N + n0 + n;
    if (n + 8 <= cols) {
      *reinterpret_cast<f16x8_any*>(dst) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < cols) dst[e] = o[e];
    }
  }
}

// n workgroups; the first dimension is a multiple of the XCDs and no dimension
// counts 2^32 threads.
dim3 grid2(int64_t n) {
  constexpr int64_t X = 1 << 21;
  return n <= X ? dim3((uint32_t)n) : dim3((uint32_t)X, (uint32_t)((n + X - 1) / X));
}

// Dynamic LDS above 64 KB has to be allowed once a device.
template <class C, bool ALIGNED, bool GELU>
hipError_t allow_lds() {
  static std::atomic<uint64_t> done{0};
  if (C::LDS <= 64 * 1024) return hipSuccess;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_i8_kernel<C, ALIGNED, GELU>),
                          hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <class C, bool ALIGNED, bool GELU>
hipError_t launch(const Args& g, hipStream_t s) {
  const hipError_t e = allow_lds<C, ALIGNED, GELU>();
  if (e != hipSuccess) return e;
  const int tm = (g.M - 1) / C::BM + 1, tn = (g.N - 1) / C::BN + 1;
  const int64_t items = (int64_t)tm * tn;
  if (items > INT32_MAX / 2) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_i8_kernel<C, ALIGNED, GELU>),
                     grid2((items + kXcds - 1) / kXcds * kXcds), dim3(C::THREADS), C::LDS, s, g, tm,
                     tn);
  return hipGetLastError();
}

template <class C>
hipError_t launch(const Args& g, bool aligned, bool gelu, hipStream_t s) {
  if (aligned) return gelu ? launch<C, true, true>(g, s) : launch<C, true, false>(g, s);
  return gelu ? launch<C, false, true>(g, s) : launch<C, false, false>(g, s);
}

}  // namespace

hipError_t gemm_i8(const int8_t* A, const float* sa, const int8_t* B, const float* sb,
                   const f16* bias, f16* C, int M, int N, int K, bool gelu, hipStream_t s) {
  const Args g{A, B, sa, sb, bias, C, M, N, K};
  const bool aligned = K % kChunk == 0 && (((uintptr_t)A | (uintptr_t)B) & 15) == 0;
  const int64_t t128 = (int64_t)((M - 1) / 128 + 1) * ((N - 1) / 128 + 1);
  if (t128 >= 128) return launch<Cfg<128, 128, 2, 2, 1, 3>>(g, aligned, gelu, s);
  return launch<Cfg<32, 64, 1, 2, 4, 2>>(g, aligned, gelu, s);
}

}  // namespace bbh

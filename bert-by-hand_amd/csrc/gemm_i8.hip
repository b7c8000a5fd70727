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
// Bounds, measured on MI355X: large products the clock that power leaves the
// matrix cores, and that they idle a third of its cycles (8192^3 440-470 us, 2.3-2.5
// POP/s, 66% busy at 1.65-1.7 GHz; independent products on random codes reach 3.48,
// always busy at that clock): a slice's copies take as long as its products, and
// with two slots they are asked for in one burst after each barrier; few rows
// against many the waits of a workgroup's three steps a slice more than the reading
// of B (64 x 200003 x 384 25.7 us, 4.0 TB/s with its output, of a new index each time;
// 18.4 of the same one, from the memory-side cache in part), as each of the 64 x 64
// tiles copies A again; a short K its copies from L2, epilogue and stores in turn
// (8192 x 1536 x 384 with GELU 14.0 us); the smallest a launch and one latency (16 x
// 1536 x 384 3.0 us, 1 x 4096 x 4096 5.6).
//
// K goes in slices of 128 bytes: a row of a slice is one cache line, eight
// 16-byte chunks, and logical chunk c of row r sits in slot c ^ ((r >> 1) & 7)
// (the layout of pipe.h's 64-wide fp16 slice, byte for byte).

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "int8.h"
#include "pipe.h"

namespace bbh {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef f16x8 f16x8_any __attribute__((aligned(2)));

constexpr int kSlice = 128;  // bytes of K a slice
constexpr int kChunk = 16;
constexpr int64_t kXcdL2 = 4 << 20;  // bytes of an XCD's L2

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
  return to_half(GELU ? gelu_wide(v) : v);
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
  static constexpr int MB = BM < 32 ? 16 : 32;                // matrix block MB x MB
  static constexpr int KB = MB == 16 ? 64 : 32, STEPS = kSlice / KB;  // bytes of K a product
  static constexpr int NV = MB * MB / 64;                     // sums a lane a block
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / MB, FN = TN / MB;
  static constexpr int LA = BM / 8 / GW, LB = BN / 8 / GW, L = LA + LB;  // 1 KB copies a wavefront
  static constexpr int STAGE = (BM + BN) * kSlice;
  static constexpr int RING = STAGE * R * KS;
  static constexpr int OUT_LD = BN + 8;  // padded row of the fp16 tile (KS == 1)
  static constexpr int SUM_LD = BN + 4;  // of the groups' int32 tiles
  static constexpr int OUT = KS == 1 ? BM * OUT_LD * 2 : KS * BM * SUM_LD * 4;
  static constexpr int VEC = RING > OUT ? RING : OUT;       // sa, sb, bias follow
  static constexpr int LDS = VEC + (BM + 2 * BN) * 4;
  static constexpr int CH = (BM + BN) * 8 / (64 * GW);      // chunks a thread (last slice)
  static_assert(TM % MB == 0 && TN % MB == 0, "whole blocks");
  static_assert(BM % (8 * GW) == 0 && BN % (8 * GW) == 0, "a copy is of one operand");
  static_assert(R >= 1 && (R - 1) * L < 64, "vmcnt range");
  static_assert(STEPS == 2 || STEPS == 4, "K steps");
  static_assert(BM <= THREADS && BN <= THREADS, "a thread loads one of each vector");
  static_assert(LDS <= (int)kLdsMax && THREADS <= 1024, "workgroup");
};

// Copies of this wavefront's share of a slice: global -> LDS, 1 KB = 8 rows a
// copy.  Rows and bytes past the operand are out of the resource's bounds, as
// is everything at an offset of kNowhere: such copies read no memory and write
// zeros.
constexpr uint32_t kNowhere = 1u << 30;
__device__ __forceinline__ uint32_t head(const int8_t* p) { return (uint32_t)(uintptr_t)p & 3; }
struct Copier {
  __amdgpu_buffer_rsrc_t src;
  uint32_t lane[2], step;  // byte offset in an even / odd block of 8 rows; 8 rows
  __device__ __forceinline__ Copier(const int8_t* base, int rows, int K)
      : src(buffer_of(base - head(base), (head(base) + (uint32_t)rows * K + 3) & ~3u)),
        step(8u * K) {
    const int l = threadIdx.x & 63, r = l >> 3;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      lane[p] = ((head(base) + r * K) & ~3u) + (((l & 7) ^ (p << 2 | r >> 1)) << 4);
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

template <int MB>
struct Product;
template <>
struct Product<32> {
  typedef i32x16 Acc;
  __device__ static __forceinline__ Acc mul(i32x4 b, i32x4 a, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(b, a, c, 0, 0, 0);
  }
};
template <>
struct Product<16> {
  typedef i32x4 Acc;
  __device__ static __forceinline__ Acc mul(i32x4 b, i32x4 a, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, c, 0, 0, 0);
  }
};

// Operands of one K step: lane l holds 16 bytes of row l % MB, chunk l / MB of
// the step's, of each block.  A product gives it the columns 8 q + 4 (l / MB)
// .. + 3, q = 0 .. NV / 4 - 1, of row l % MB.
template <class C, bool SHIFTED>
struct Frags {
  i32x4 a[C::FM], b[C::FN];
  static constexpr bool BEFORE = SHIFTED && C::MB == 16;
  int pa[BEFORE ? C::FM : 1] = {}, pb[BEFORE ? C::FN : 1] = {};  // the dwords before (Carry)
  __device__ static __forceinline__ int lane_at(int lane) {
    const int r = lane % C::MB;
    return r * kSlice + ((lane / C::MB ^ (r >> 1 & 7)) << 4);
  }
  // kShifted: where a lane finds the dword before its chunk: in the chunk before
  // of the same step, or, for the step's first chunk, in the last chunk of the
  // step before.  So the lanes of the first read the last one's, for the step
  // that follows (Carry).
  __device__ static __forceinline__ int lane_before(int lane) {
    const int r = lane % C::MB, c = lane / C::MB, last = 64 / C::MB - 1;
    return r * kSlice + (((c ? c - 1 : last) ^ (r >> 1 & 7)) << 4) + 12;
  }
  __device__ __forceinline__ void read(const char* st, int j, int at, int before, int wm, int wn) {
    const char* p = st + (at ^ (j * C::KB));
#pragma unroll
    for (int f = 0; f < C::FM; ++f)
      a[f] = *reinterpret_cast<const i32x4*>(p + (wm * C::TM + f * C::MB) * kSlice);
#pragma unroll
    for (int f = 0; f < C::FN; ++f)
      b[f] = *reinterpret_cast<const i32x4*>(p + (C::BM + wn * C::TN + f * C::MB) * kSlice);
    if constexpr (BEFORE) {
      const char* e = st + (before ^ (j * C::KB));
#pragma unroll
      for (int f = 0; f < C::FM; ++f)
        pa[f] = *reinterpret_cast<const int*>(e + (wm * C::TM + f * C::MB) * kSlice);
#pragma unroll
      for (int f = 0; f < C::FN; ++f)
        pb[f] = *reinterpret_cast<const int*>(e + (C::BM + wn * C::TN + f * C::MB) * kSlice);
    }
  }
  __device__ __forceinline__ void mul(typename Product<C::MB>::Acc (&acc)[C::FM][C::FN]) const {
#pragma unroll
    for (int fm = 0; fm < C::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < C::FN; ++fn)
        acc[fm][fn] = Product<C::MB>::mul(b[fn], a[fm], acc[fm][fn]);
  }
};

// kShifted: of the 20 raw bytes that end with a lane's chunk, the 16 from byte
// `sa` (or `sb`) on are its bytes of K.  The first four are the last of the chunk
// before: that of the lane MB below, or, for the step's first chunk, of the
// step before, kept here.  With MB = 32 both come from one exchange of the
// wavefront's halves; with 16 the dword is read from LDS (with 32, too, that took
// the LDS half as long again as the chunks do).
template <class C>
struct Carry {
  int a[C::FM], b[C::FN];
  uint32_t sa, sb;
  bool first;  // of the step's chunks
  __device__ __forceinline__ void one(i32x4& v, int& keep, int before, uint32_t by) const {
    int p;
    if constexpr (C::MB == 32) {
      const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)keep, (uint32_t)v[3], false, false);
      p = (int)(first ? h[1] : h[0]);
      keep = v[3];
    } else {
      p = first ? keep : before;
      keep = before;
    }
    v[3] = __builtin_amdgcn_alignbyte(v[3], v[2], by);
    v[2] = __builtin_amdgcn_alignbyte(v[2], v[1], by);
    v[1] = __builtin_amdgcn_alignbyte(v[1], v[0], by);
    v[0] = __builtin_amdgcn_alignbyte(v[0], p, by);
  }
  __device__ __forceinline__ void shift(Frags<C, true>& f) {
    constexpr bool B = Frags<C, true>::BEFORE;
#pragma unroll
    for (int i = 0; i < C::FM; ++i) one(f.a[i], a[i], f.pa[B ? i : 0], sa);
#pragma unroll
    for (int i = 0; i < C::FN; ++i) one(f.b[i], b[i], f.pb[B ? i : 0], sb);
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

// How slices reach the ring: by buffer loads to LDS, 16 bytes a lane, which need
// 4-byte alignment only.
//  kCopies   K % 16 == 0, 16-byte aligned operands.
//  kCopies4  K % 4 == 0, 4-byte aligned operands: whole slices; the last part of K,
//            whose chunks would cross a row's end, goes through registers.
//  kShifted  any K and address: a row's raw bytes from the 4-byte boundary at or
//            before its first, and again the last part through registers.  Bytes
//            of K come from the raw ones by a shift that is the lane's own, as
//            its rows are equal modulo 4 (Carry): slice s holds k = 128 s - 4 ..
//            128 s + 123.  Only dwords that hold a byte of the operand are read,
//            and what else they hold is cleared in A before the product.
// 4000 x 4000 x 2001 49 us, 2004 43, 2000 40 (through registers altogether 65);
// 2003 x 1111 x 777 10.9, 780 9.6, 768 8.4 (12.4).
enum Feed { kCopies, kCopies4, kShifted };

template <class C, int FEED, bool GELU>
__global__ __launch_bounds__(C::THREADS) void gemm_i8_kernel(Args g, int tm, int tn) {
  extern __shared__ __align__(16) char smem[];
  constexpr bool SHIFTED = FEED == kShifted;
  constexpr bool TAIL = FEED != kCopies;  // the last slice goes through registers
  static_assert(!TAIL || C::R > 1, "a ring of one slice has whole slices only");
  int bm, bn;
  if (!tile_of(tm, tn, bm, bn)) return;
  const int K = g.K, m0 = bm * C::BM, n0 = bn * C::BN;
  const int rows = min(C::BM, g.M - m0), cols = min(C::BN, g.N - n0);
  const int8_t* A = g.A + (size_t)m0 * K;
  const int8_t* B = g.B + (size_t)n0 * K;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int grp = wave / C::GW, w = wave % C::GW, wm = w / C::WN, wn = w % C::WN;

  // The epilogue's vectors: loaded here, ahead of the copies, and put into LDS
  // after the K loop, so that nothing waits for them.
  const int tid = threadIdx.x;
  float hsa = 0.f, hsb = 0.f;
  f16 hbias = 0.f;
  if (tid < rows) hsa = g.sa[m0 + tid];
  if (tid < cols) {
    hsb = g.sb[n0 + tid];
    if (g.bias) hbias = g.bias[n0 + tid];
  }

  typename Product<C::MB>::Acc acc[C::FM][C::FN];
#pragma unroll
  for (int fm = 0; fm < C::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < C::FN; ++fn)
#pragma unroll
      for (int i = 0; i < C::NV; ++i) acc[fm][fn][i] = 0;

  // Iteration i of a group is slice i * KS + grp.  Every group has `even` whole
  // slices; then one iteration more, in which a group has a whole slice, the
  // last part of K or none, unless no group has any.
  const int full = (SHIFTED ? K + 3 : K) / kSlice;
  const int total = SHIFTED ? full + 1 : full + (K % kSlice ? 1 : 0);
  const int even = full / C::KS, iters = (total + C::KS - 1) / C::KS;
  char* const ring = smem + grp * C::R * C::STAGE;
  char* const ring_end = ring + C::R * C::STAGE;
  const Copier ca(A, rows, K), cb(B, cols, K);
  auto slice = [&](int i) {
    if constexpr (SHIFTED && C::KS > 1)  // a group's are next to each other
      return i < even ? grp * even + i : i > even ? total : C::KS * even + grp;
    else
      return i * C::KS + grp;
  };
  auto issue = [&](int i, char* dst) {  // the slice of iteration i into a slot
    const int s = slice(i);
    const uint32_t at = s < (TAIL ? full : total) ? (uint32_t)s * kSlice : kNowhere;
    ca.template copy<C::LA>(at, dst, w);
    cb.template copy<C::LB>(at, dst + C::BM * kSlice, w);
  };
  // The last slice through registers.  Chunk j of a thread is a row of A or of B by
  // j alone; rows past the tile's last are that one again (nothing of theirs is
  // written).
  constexpr int CH = TAIL ? C::CH : 1;
  i32x4 held[CH];
  auto load = [&] {
    if (slice(even) != full) return;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int r = w * 8 + (lane >> 3) + j * 8 * C::GW, k = full * kSlice + (lane & 7) * kChunk;
      const int8_t* row = j * 8 * C::GW < C::BM ? A + (uint32_t)min(r, rows - 1) * K
                                                : B + (uint32_t)min(r - C::BM, cols - 1) * K;
      const int8_t* p = row - (SHIFTED ? head(row) : 0) + k;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        held[j][e] = p + 4 * e < row + K ? reinterpret_cast<const int*>(p)[e] : 0;
    }
  };
  auto put = [&](char* dst) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int r = w * 8 + (lane >> 3) + j * 8 * C::GW;
      *reinterpret_cast<i32x4*>(dst + r * kSlice + (((lane & 7) ^ (r >> 1 & 7)) << 4)) = held[j];
    }
  };
  auto next = [&](char* p) { return p + C::STAGE == ring_end ? ring : p + C::STAGE; };
  char* slot = ring;      // of the slice that is read
  char* refill = ring;    // the slot that the next copies go to

  typedef Frags<C, SHIFTED> F;
  const int at = F::lane_at(lane), lrow = lane % C::MB, lchunk = lane / C::MB;
  const int before = SHIFTED ? F::lane_before(lane) : 0;
  Carry<C> carry{}, later{};
  auto carry_into = [&](int s, Carry<C>& c) {  // 0 < s <= full
#pragma unroll
    for (int f = 0; f < C::FM; ++f) {
      const int8_t* row = A + (size_t)min(wm * C::TM + f * C::MB + lrow, rows - 1) * K;
      c.a[f] = *reinterpret_cast<const int*>(row - head(row) + s * kSlice - 4);
    }
#pragma unroll
    for (int f = 0; f < C::FN; ++f) {
      const int8_t* row = B + (size_t)min(wn * C::TN + f * C::MB + lrow, cols - 1) * K;
      c.b[f] = *reinterpret_cast<const int*>(row - head(row) + s * kSlice - 4);
    }
  };
  if constexpr (SHIFTED) {
    carry.sa = later.sa = head(A + lrow * (K & 3));
    carry.sb = later.sb = head(B + lrow * (K & 3));
    carry.first = later.first = lchunk == 0;
    if constexpr (C::KS > 1) {
      if (even > 0 && grp > 0) carry_into(grp * even, carry);
      if (slice(even) > 0 && slice(even) <= full) carry_into(slice(even), later);
    }
  }
  if (!TAIL || full > 0) {
#pragma unroll
    for (int i = 0; i < C::R; ++i) issue(i, ring + i * C::STAGE);
  }
  // Makes slice i readable: its copies have landed (those of later ones may be
  // in flight: R - 1 slices behind the first, then R - 2, as the next copies come
  // after this), and every wavefront has read slice i - 1, whose slot the next
  // copies fill.
  auto arrive = [&](auto first) {
    wait_vm<(C::R - (decltype(first)::value || C::R == 1 ? 1 : 2)) * C::L>();
    lds_barrier();
  };
  constexpr std::true_type kFirst{};
  constexpr std::false_type kLater{};
  auto advance = [&](int i) {  // the copies that follow arrive() of slice i
    if constexpr (C::R > 1) {
      issue(i + C::R - 1, refill);
      refill = next(refill);
    }
  };
  auto reload = [&](int i) {  // R == 1: the next slice over this one
    if constexpr (C::R == 1) {
      lds_barrier();
      issue(i, ring);
    }
  };
  F f0, f1;
  auto mul = [&](F& f) {
    if constexpr (SHIFTED) carry.shift(f);
    f.mul(acc);
  };
  // kShifted: the bytes before the first of K
  auto clear_head = [&](int s) {
    if (SHIFTED && s == 0 && lchunk == 0)
#pragma unroll
      for (int f = 0; f < C::FM; ++f) f0.a[f][0] &= (int)(~0u << (8 * carry.sa));
  };
  constexpr int RD = C::FM + C::FN, MF = C::FM * C::FN;
  // All K steps of the slice but the last, each beside the reads of the next.
  auto most = [&] {
    __builtin_amdgcn_sched_barrier(0);
    f1.read(slot, 1, at, before, wm, wn);
    mul(f0);
    interleave<RD, MF>();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (C::STEPS == 4) {
      f0.read(slot, 2, at, before, wm, wn);
      mul(f1);
      interleave<RD, MF>();
      __builtin_amdgcn_sched_barrier(0);
      f1.read(slot, 3, at, before, wm, wn);
      mul(f0);
      interleave<RD, MF>();
      __builtin_amdgcn_sched_barrier(0);
    }
    slot = next(slot);
  };
  auto step = [&](int i) {
    most();
    reload(i);
    arrive(kLater);
    f0.read(slot, 0, at, before, wm, wn);
    advance(i);
    mul(f1);
    interleave<RD, MF>();
  };
  if (even > 0) {
    arrive(kFirst);
    f0.read(slot, 0, at, before, wm, wn);
    clear_head(slice(0));
    for (int i = 1; i < even; ++i) step(i);
    if constexpr (TAIL) load();
    most();
    if (C::R == 1 && iters > even) reload(even);
    mul(f1);
  } else if constexpr (TAIL) {
    load();
  }
  if (iters > even) {
    if constexpr (TAIL) {
      // A copy from nowhere still writes its slot (zeros): every wavefront's have
      // landed before any puts what belongs there.
      if (full > 0) {
        wait_vm<0>();
        lds_barrier();
      }
      if (slice(even) == full) put(slot);
    }
    if (even == 0)
      arrive(kFirst);
    else
      arrive(kLater);
    // kShifted: a slice's k begin 4 before its raw bytes
    const int s = slice(even), left = min(kSlice, K - s * kSlice + (SHIFTED ? 4 : 0));
    if constexpr (SHIFTED && C::KS > 1) carry = later;
    for (int j = 0; j * C::KB < left; ++j) {
      f0.read(slot, j, at, before, wm, wn);
      // past K: the next row's bytes in both operands, cleared in one
      if (FEED == kCopies && j * C::KB + lchunk * kChunk >= left)
#pragma unroll
        for (int f = 0; f < C::FM; ++f) f0.a[f] = i32x4{0, 0, 0, 0};
      if constexpr (SHIFTED) {
        if (j == 0) clear_head(s);
        carry.shift(f0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = left - j * C::KB - lchunk * kChunk - 4 * e;  // bytes of this dword in K
          const int keep = n >= 4 ? -1 : n <= 0 ? 0 : (int)((1u << (8 * n)) - 1);
#pragma unroll
          for (int f = 0; f < C::FM; ++f) f0.a[f][e] &= keep;
        }
      }
      f0.mul(acc);
    }
  }
  float* vsa = reinterpret_cast<float*>(smem + C::VEC);
  float* vsb = vsa + C::BM;
  float* vbias = vsb + C::BN;
  if (tid < C::BM) vsa[tid] = hsa;
  if (tid < C::BN) {
    vsb[tid] = hsb;
    vbias[tid] = (float)hbias;
  }
  wait_vm<0>();  // copies from nowhere are still copies
  lds_barrier();  // the ring is free

  if constexpr (C::KS == 1) {
    f16* tile = reinterpret_cast<f16*>(smem);
#pragma unroll
    for (int fm = 0; fm < C::FM; ++fm) {
      const int m = wm * C::TM + fm * C::MB + lrow;
      const float sa = vsa[m];
#pragma unroll
      for (int fn = 0; fn < C::FN; ++fn)
#pragma unroll
        for (int q = 0; q < C::NV / 4; ++q) {
          const int n = wn * C::TN + fn * C::MB + 8 * q + 4 * lchunk;
          const f32x4 sb = *reinterpret_cast<const f32x4*>(vsb + n);
          const f32x4 bi = *reinterpret_cast<const f32x4*>(vbias + n);
          f16x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = finish<GELU>(acc[fm][fn][4 * q + e], sa, sb[e], bi[e]);
          *reinterpret_cast<f16x4*>(tile + m * C::OUT_LD + n) = o;
        }
    }
  } else {
    int* sums = reinterpret_cast<int*>(smem) + grp * C::BM * C::SUM_LD;
#pragma unroll
    for (int fm = 0; fm < C::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < C::FN; ++fn)
#pragma unroll
        for (int q = 0; q < C::NV / 4; ++q) {
          const int m = wm * C::TM + fm * C::MB + lrow;
          const int n = wn * C::TN + fn * C::MB + 8 * q + 4 * lchunk;
          *reinterpret_cast<i32x4*>(sums + m * C::SUM_LD + n) =
              i32x4{acc[fm][fn][4 * q], acc[fm][fn][4 * q + 1], acc[fm][fn][4 * q + 2],
                    acc[fm][fn][4 * q + 3]};
        }
  }
  lds_barrier();
  // Eight columns a thread at a time, 16-byte stores.
  auto chunk = [&](int m, int n) {
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
    return o;
  };
  constexpr int CPR = C::BN / 8, N8 = C::BM * CPR;  // chunks a row, a tile
  f16* const out = g.C + (size_t)m0 * g.N + n0;
  if (N8 % C::THREADS == 0 && rows == C::BM && cols == C::BN) {
    // a whole tile: up to four reads in flight before their stores
    constexpr int IT = N8 >= C::THREADS ? N8 / C::THREADS : 1, U = IT % 4 == 0 ? 4 : 1;
    const int m = tid / CPR, n = tid % CPR * 8;
    auto write = [&](auto stream) {
      f16* dst = out + (size_t)m * g.N + n;
#pragma unroll
      for (int i = 0; i < IT; i += U) {
        f16x8 o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) o[u] = chunk(m + (i + u) * (C::THREADS / CPR), n);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          f16x8_any* p = reinterpret_cast<f16x8_any*>(dst);
          if constexpr (decltype(stream)::value)
            __builtin_nontemporal_store(o[u], p);
          else
            *p = o[u];
          dst += (size_t)(C::THREADS / CPR) * g.N;
        }
      }
    };
    // An output beyond an XCD's L2 is written past it, where it would displace the
    // operands that other tiles read again: 8192 x 1536 x 384 with GELU 15.9 -> 13.6
    // us, 131072 x 384 x 384 47.9 -> 38.3, 2048 x 1536 x 384 6.5 -> 6.2 (inputs that
    // change from call to call; the same ones again 14.9 -> 14.0, 38.6 -> 40.2, 5.9 both);
    // but 512 x 1536 x 384 with the quantising that reads it 8.0 -> 8.2, and tiles of
    // 256 x 256, whose operands are read less often, 51.8 -> 55.8 (8192 x 4096 x 1024).
    // Only in rows of whole lines: L2 puts the parts of others together, which past
    // it are written one by one (64 x 1000003 x 128 60 -> 119, 64 x 200003 x 384 25.7
    // -> 31.0, 18.4 -> 21.5 with the same index again).
    // (The comments in the assembly keep the compiler from merging the two, which
    // would make every store an ordinary one.)
    const int64_t written = (int64_t)g.M * g.N * 2;
    const bool lines = ((uintptr_t)g.C | (uint32_t)g.N * 2) % 128 == 0;
    if (C::BM * C::BN < 256 * 256 && written >= kXcdL2 && lines) {
      asm volatile("; past L2" ::: "memory");
      write(std::true_type{});
      asm volatile("; end past L2" ::: "memory");
    } else {
      write(std::false_type{});
    }
    return;
  }
  for (int i = tid; i < N8; i += C::THREADS) {
    const int m = i / CPR, n = i % CPR * 8;
    if (m >= rows || n >= cols) continue;
    const f16x8 o = chunk(m, n);
    f16* dst = out + (size_t)m * g.N + n;
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
template <class C, int FEED, bool GELU>
hipError_t allow_lds() {
  static std::atomic<uint64_t> done{0};
  if (C::LDS <= 64 * 1024) return hipSuccess;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_i8_kernel<C, FEED, GELU>),
                          hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <class C, int FEED, bool GELU>
hipError_t launch(const Args& g, hipStream_t s) {
  const hipError_t e = allow_lds<C, FEED, GELU>();
  if (e != hipSuccess) return e;
  const int tm = (g.M - 1) / C::BM + 1, tn = (g.N - 1) / C::BN + 1;
  const int64_t items = (int64_t)tm * tn;
  if (items > INT32_MAX / 2) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_i8_kernel<C, FEED, GELU>),
                     grid2((items + kXcds - 1) / kXcds * kXcds), dim3(C::THREADS), C::LDS, s, g, tm,
                     tn);
  return hipGetLastError();
}

template <class C, int FEED>
hipError_t run(const Args& g, bool gelu, hipStream_t s) {
  return gelu ? launch<C, FEED, true>(g, s) : launch<C, FEED, false>(g, s);
}

// The tiles, and what one costs a CU in cycles: a byte of K costs the larger of
// its operand bytes at 32 a cycle, which is what the copies sustain from L2 (44
// where many single-wavefront workgroups share a CU), and `mfma`, the measured
// pace of the tile's products; `fixed` is the rest of a tile's time (first
// copies, epilogue) that other workgroups on the CU do not hide.  The tile
// whose ceil(tiles / CUs) rounds cost least is launched.
struct Tile {
  int bm, bn;
  float mfma, fixed;
};
constexpr Tile kTiles[] = {{256, 256, 22.f, 11400.f}, {256, 128, 15.8f, 4000.f},
                           {128, 128, 8.6f, 1000.f},  {64, 128, 4.4f, 2000.f},
                           {128, 64, 5.4f, 2200.f},   {64, 64, 2.3f, 500.f},
                           {32, 64, 1.2f, 600.f},     {32, 32, 0.7f, 900.f},
                           {16, 32, 0.5f, 1500.f},    {16, 16, 0.3f, 120.f}};
constexpr int kCus = kXcds * kXcdCus;
int64_t rounds_of(const Tile& t, int M, int N) {
  const int64_t n = (int64_t)((M - 1) / t.bm + 1) * ((N - 1) / t.bn + 1);
  return (n + kCus - 1) / kCus;
}

int pick_tile(int M, int N, int K) {
  int best = -1;
  float least = 0.f;
  for (int i = 0; i < (int)(sizeof kTiles / sizeof kTiles[0]); ++i) {
    const Tile& t = kTiles[i];
    const int64_t rounds = rounds_of(t, M, N);
    // rows past M and N are not read
    const float copies = (float)(std::min(M, t.bm) + std::min(N, t.bn)) /
                         (t.bn == 16 && rounds > 2 ? 44.f : 32.f);
    const float cost = (float)rounds * ((float)K * (copies > t.mfma ? copies : t.mfma) + t.fixed);
    if (best < 0 || cost < least) {
      least = cost;
      best = i;
    }
  }
  return best;
}

template <int FEED>
hipError_t dispatch(const Args& g, bool gelu, hipStream_t s) {
  const int K = g.K, t = pick_tile(g.M, g.N, K);
  // One round, a workgroup a CU, and a long K: nothing but its own copies hides
  // a workgroup's waits, so it has more of them in flight (or more groups).
  const int64_t rounds = rounds_of(kTiles[t], g.M, g.N);
  const bool alone = rounds == 1 && K >= 1024;
  // Tiles of 16 x 16 by one wavefront a workgroup: where K is short (16 x 1536 x
  // 384 2.7 us against 3.1) or there are many, not too long each (8 x 33206 x 2704
  // 17.0 against 19.7, but 1 x 32000 x 4096 31.5 against 27.6).
  const bool one_wave = K <= 512 || (rounds >= 8 && K < 4096);
  // Several rounds: a ring of one slice, so that twice the workgroups share a CU
  // and hide each other's copies and epilogues (128 x 128 tiles, 16388 x 3190 x 368
  // 41.2 us against 43.9 with two, 44705 x 1024 x 800 58.3 and 62.1), until a long
  // K leaves little to hide (4004 x 3648 x 4240 98.2 and 86.9); smaller tiles only
  // where K is short (64 x 128, 18842 x 512 x 256 7.5 and 9.0, but 4749 x 1984 x
  // 3488 60.8 and 58.6).  Where the last slice goes through registers a second
  // slice hides that better (4000 x 4000 x 2004 52.0 and 50.0, 5336 x 3392 x 1969
  // 77.0 and 67.5).
  if constexpr (FEED == kCopies) {
    if (rounds > 1 && K < 4096) {
      if (t == 2) return run<Cfg<128, 128, 4, 2, 1, 1>, FEED>(g, gelu, s);
      if (t == 3 && K <= 512) return run<Cfg<64, 128, 1, 4, 1, 1>, FEED>(g, gelu, s);
      if (t == 5 && K <= 512) return run<Cfg<64, 64, 2, 2, 1, 1>, FEED>(g, gelu, s);
      if (t == 6 && K <= 512) return run<Cfg<32, 64, 1, 2, 1, 1>, FEED>(g, gelu, s);
    }
  }
  switch (t) {
    case 0: return run<Cfg<256, 256, 2, 4, 1, 2>, FEED>(g, gelu, s);
    case 1: return run<Cfg<256, 128, 4, 2, 1, 3>, FEED>(g, gelu, s);
    case 2:
      return alone ? run<Cfg<128, 128, 2, 4, 1, 3>, FEED>(g, gelu, s)
                   : run<Cfg<128, 128, 4, 2, 1, 2>, FEED>(g, gelu, s);
    case 3:
      return alone ? run<Cfg<64, 128, 2, 2, 1, 3>, FEED>(g, gelu, s)
                   : run<Cfg<64, 128, 1, 4, 1, 2>, FEED>(g, gelu, s);
    case 4:
      return alone ? run<Cfg<128, 64, 2, 2, 1, 3>, FEED>(g, gelu, s)
                   : run<Cfg<128, 64, 2, 2, 1, 2>, FEED>(g, gelu, s);
    case 5:
      return alone                      ? run<Cfg<64, 64, 2, 2, 2, 3>, FEED>(g, gelu, s)
             : rounds == 2 && K >= 1024 ? run<Cfg<64, 64, 2, 2, 1, 3>, FEED>(g, gelu, s)
                                        : run<Cfg<64, 64, 2, 2, 1, 2>, FEED>(g, gelu, s);
    case 6:
      return rounds > 2 ? run<Cfg<32, 64, 1, 2, 1, 2>, FEED>(g, gelu, s)
                        : run<Cfg<32, 64, 1, 2, 2, 3>, FEED>(g, gelu, s);
    case 7:
      return alone                    ? run<Cfg<32, 32, 1, 1, 4, 4>, FEED>(g, gelu, s)
             : K <= 512 || rounds > 2 ? run<Cfg<32, 32, 1, 1, 1, 2>, FEED>(g, gelu, s)
                                      : run<Cfg<32, 32, 1, 1, 4, 2>, FEED>(g, gelu, s);
    case 8: return run<Cfg<16, 32, 1, 1, 4, 4>, FEED>(g, gelu, s);
    default:
      // (Shifting takes a wavefront's time, so fewer slices each: 5 x 384 x 9677 7.3 us
      // with eight groups, 8.9 with four; 2 x 148 x 2227 4.8 and 5.1.)
      if constexpr (FEED == kShifted)
        if (rounds == 1 && K > 1536) return run<Cfg<16, 16, 1, 1, 8, 2>, FEED>(g, gelu, s);
      return one_wave    ? run<Cfg<16, 16, 1, 1, 1, 2>, FEED>(g, gelu, s)
             : K <= 1536 ? run<Cfg<16, 16, 1, 1, 2, 2>, FEED>(g, gelu, s)
                         : run<Cfg<16, 16, 1, 1, 4, 4>, FEED>(g, gelu, s);
  }
}

}  // namespace

hipError_t gemm_i8(const int8_t* A, const float* sa, const int8_t* B, const float* sb,
                   const f16* bias, f16* C, int M, int N, int K, bool gelu, hipStream_t s) {
  const Args g{A, B, sa, sb, bias, C, M, N, K};
  const uintptr_t at = (uintptr_t)A | (uintptr_t)B | (uintptr_t)K;
  return at % 16 == 0  ? dispatch<kCopies>(g, gelu, s)
         : at % 4 == 0 ? dispatch<kCopies4>(g, gelu, s)
                       : dispatch<kShifted>(g, gelu, s);
}

}  // namespace bbh

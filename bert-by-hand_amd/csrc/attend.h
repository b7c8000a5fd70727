// Host launchers of rotary positions (rope.hip) and of attention for models
// other than MiniLM (attend.hip).  As in kernels.h each enqueues on `s` and
// returns the launch status; the argument checks are in capi_attend.hip.
#pragma once

#include "common.h"

namespace bbh {

// A tensor of heads: element (b, i, h, d) at data[b * batch + i * row + h * head + d].
struct Heads {
  int64_t batch, row, head;
};

struct Divisor {
  uint32_t hi, lo;  // ceil(2^64 / d); 0: d is 1
};

// Largest cap under which scores are computed from 1 / (1 + e^2x) and its constant left out
// (attend.hip, shape()).
constexpr float kNearCap = 128.f;

struct AttendParams {
  const f16 *q, *k, *v;
  f16* out;
  Heads qs, ks, vs, os;
  const int32_t *q_offsets, *k_offsets, *q_lengths, *k_lengths, *prefix, *mask;
  const float *slopes, *table;
  float* part_o;   // partial outputs of a split call: (row slot, split, HD) fp32
  float2* part_ml;  // and their (maximum, sum)
  int64_t q_rows, k_rows;
  int b0;  // first sequence of a launch
  int batch, q_len, k_len, heads, kv_heads, dim, group;
  Divisor by_cols, by_splits, by_kv;  // blocks * splits, splits, kv_heads
  uint32_t group_magic;  // ceil(2^32 / group), or 0
  int left, right, half;
  float mscale;      // scores times this are powers of two: scale, twice a cap or a cap, each * log2(e)
  float lag;         // how far above a row's maximum its scores may lie before that is raised (attend.hip)
  float bias_scale;  // log2(e) / mscale: biases in the units of the scores
  bool table_lds;    // the table fits beside the tiles
  float cap_k;  // 2 * log2(e) * scale / cap of a cap up to kNearCap, scale / cap of a larger one; 0: none
  bool wide_cap;
  int blocks, splits, chunk;  // row blocks; splits of a block's key tiles, `chunk` tiles each
};

constexpr int kMaxRopePairs = 128;

// Angles as fractions of a turn in 64-bit fixed point: position * step modulo 2^64
// is the angle modulo a turn, exactly, for any int32 position.
struct RopeSteps {
  uint2 step[kMaxRopePairs];  // (low, high) word of a pair's turns a position
};

struct RopeParams {
  struct Part {  // q, k or v
    const f16* x;
    f16* y;
    const f16* gamma;
    int64_t x_row, x_head, y_row, y_head;
    int heads;
  };
  Part q, k, v;
  const int32_t* positions;
  const int64_t* kv_rows;
  int64_t kv_out_rows;
  int row0, rows;  // first row of a launch, the row past its last
  int seq, dim, rot;
  bool interleaved;
  float eps, magnitude;
};

// q, k normed (where they have a gamma) and rotated, v moved; a part without heads is
// none.  rot 0: no rotation.
hipError_t rope_heads(const RopeParams& p, const RopeSteps& steps, hipStream_t s);

// Fills in blocks, splits and chunk and launches.  part_bytes: scratch at hand.
hipError_t attend(AttendParams p, void* scratch, size_t scratch_bytes, hipStream_t s);
// Bytes of scratch with which attend splits the keys as it would like to.
size_t attend_scratch(const AttendParams& p);

}  // namespace bbh

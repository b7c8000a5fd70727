/*
 * bbh_attend.h - rotary positions and attention for models other than MiniLM.
 *
 * No counterpart in the reference, whose encoder has learned absolute positions
 * and one form of attention (bbh_attention: head size 32, at most 512 tokens, a
 * key mask).  These operators are the pieces that the blocks of other embedding
 * models need beside bbh_linear and the norms: heads normed and rotated by their
 * positions, and attention with other head sizes, shared key/value heads, capped
 * scores, a bias by distance, a window, a prefix, documents packed end to end,
 * and a few queries over a cache of keys.  All conventions of bbh.h hold (device
 * pointers, fp16 data, `stream`, bbh_status, bbh_last_error; nothing allocates
 * device memory, so every call can be captured into a HIP graph).  Forward only,
 * as the rest of the engine.
 */
#ifndef BBH_ATTEND_H
#define BBH_ATTEND_H

#include "bbh.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A tensor of heads: element (b, i, h, d) is data[b*batch + i*row + h*head + d],
 * strides in elements.  Calls without a batch dimension ignore `batch`. */
typedef struct bbh_heads {
  void *data;
  int64_t batch, row, head;
} bbh_heads;

/* ---- rotary positions --------------------------------------------------------
 * The first rot_dim values of a head turn in pairs: with pair i at angle
 * t = position * f_i,
 *   a' = magnitude * (a cos t - b sin t),  b' = magnitude * (b cos t + a sin t).
 * A pair is (x_i, x_{i + rot_dim/2}), or (x_{2i}, x_{2i+1}) where interleaved.  The
 * other values of the head pass unchanged.  f_i = base^(-2i / rot_dim), scaled
 * for contexts `factor` times as long as the `original` one:
 *   LINEAR  f_i / factor
 *   BASE    base * factor^(rot_dim / (rot_dim - 2)) in place of base (rot_dim 2: as it is)
 *   RAMP    f_i (1 - r) + f_i / factor * r, r rising linearly from 0 to 1 over the
 *           pairs between those that turn `high` and `low` times over the original
 *           context: with d(n) = rot_dim ln(original / (2 pi n)) / (2 ln base), from
 *           pair floor(d(high)) to pair ceil(d(low)), both within [0, rot_dim - 1]
 *           (where they are one, the step is 0.001 pairs wide)
 *   BANDS   f_i s + f_i / factor * (1 - s), s rising linearly from 0 to 1 with the
 *           pair's turns over the original context, original * f_i / (2 pi), from `low`
 *           to `high`
 * NONE, LINEAR and BASE read neither original nor low and high. */
typedef enum bbh_rope_scaling {
  BBH_ROPE_NONE = 0,
  BBH_ROPE_LINEAR = 1,
  BBH_ROPE_BASE = 2,
  BBH_ROPE_RAMP = 3,
  BBH_ROPE_BANDS = 4
} bbh_rope_scaling;
typedef struct bbh_rope_config {
  int rot_dim;     /* even, 2 .. BBH_ROPE_MAX_DIM */
  int interleaved; /* 0 or 1 */
  int scaling;     /* bbh_rope_scaling */
  double base;     /* > 1 */
  double factor;   /* >= 1 */
  double original; /* > 0 */
  double low, high; /* 0 < low < high */
  double magnitude; /* of cos and sin; finite in fp32 */
  /* the f_i themselves (rot_dim / 2 finite values, host memory, copied), in radians
   * a position; NULL: from base and scaling */
  const double *frequencies;
} bbh_rope_config;
#define BBH_ROPE_MAX_DIM 256
/* A handle of the frequencies, in host memory only: usable on any device and by
 * any number of calls at once. */
typedef struct bbh_rope bbh_rope;
bbh_status bbh_rope_create(const bbh_rope_config *config, bbh_rope **out);
bbh_status bbh_rope_free(bbh_rope *rope);
/* The rot_dim / 2 frequencies of a handle, to host memory. */
bbh_status bbh_rope_frequencies(const bbh_rope *rope, double *out);

/* Rotates `rows` rows of q (and k, where k.data is not NULL), each with its number of
 * heads, and moves v (where v.data is not NULL) unchanged, in one pass:
 *   x = q or k head, first x * gamma / sqrt(mean(x^2) + eps) where the gamma is given
 *   (head_dim values, shared by the heads), then the rotation at positions[row].
 * Everything is computed in fp32 from exact angles (any int32 position) and rounded
 * to fp16 once.
 * q_out may be q, k_out k and v_out v (in place; v needs no move then); otherwise
 * outputs overlap nothing.  positions: (rows) int32; NULL: row % seq, of padded
 * batches (seq is not read otherwise).  kv_rows (optional, (rows) int64) puts row r of k and
 * v into row kv_rows[r] of k_out and v_out, as the slots of a cache of kv_out_rows rows:
 * a slot outside [0, kv_out_rows) is not written (padding), and no two rows may
 * share a slot.  rope may be NULL (norms alone).  rows >= 0, 1 <= head_dim <=
 * BBH_ROPE_MAX_DIM, rot_dim <= head_dim.  Fastest where head_dim is a multiple of 8,
 * rot_dim of 16, and addresses and strides are of 16 bytes. */
typedef struct bbh_rope_args {
  bbh_heads q, k, v, q_out, k_out, v_out; /* batch is not read */
  const void *q_gamma, *k_gamma;          /* (head_dim) fp16, or NULL */
  const int32_t *positions;
  const int64_t *kv_rows;
  int64_t kv_out_rows;
  int rows, seq, heads, kv_heads, head_dim;
  float eps;
} bbh_rope_args;
bbh_status bbh_rope_heads(const bbh_rope *rope, const bbh_rope_args *args, bbh_stream_t stream);

/* ---- attention ---------------------------------------------------------------
 * For each sequence b, query i and head h (its keys and values those of head
 * h / (heads / kv_heads)):
 *   s_j = scale * <q_i, k_j>;  cap > 0: s_j = cap * tanh(s_j / cap)
 *   s_j += table[h][clamp(j - p, -table_half, table_half) + table_half]   (table)
 *   s_j -= slopes[h] * |j - p|                                            (slopes)
 *   out_i = sum_j softmax_j(s) v_j over the keys that the query sees.
 * p = i + n_k - n_q is the query's position among the n_k keys: the last query
 * stands at the last key.  Query i sees key j < n_k if mask[b][j] != 0 (mask) and
 *   j < prefix[b], or -left <= j - p <= right  (a negative left or right: no bound).
 * right = 0 is causal.  A query that sees nothing gets zeros.
 *
 * Sequences lie in rows of q / out and k / v:
 *  - padded: b starts at b * batch elements, n_q = q_len (or q_lengths[b] where
 *    given, at most q_len), n_k = k_len (k_lengths[b]);
 *  - packed: b owns rows q_offsets[b] .. q_offsets[b+1]-1 of q_rows rows (k_offsets,
 *    k_rows), at most q_len (k_len) of them, and at most q_lengths[b] where given.
 *    Offsets outside the rows are clamped to them.
 * q and k choose separately: packed new tokens over a padded cache, say.  Rows of out
 * behind a sequence's n_q are left as they were.  Keys that no query sees (behind n_k,
 * with a mask of 0, outside of every window and the prefix) have no effect whatever they
 * hold; a value that some query sees must be finite, or may reach the others (its weight
 * there is 0, and 0 times infinity is not).
 *
 * Scores, softmax and sums are fp32; the weights are rounded to fp16 for the product
 * with v (to 2^-11 of a weight, or 2^-32 of the row's largest where that is more), the
 * output once.  Offsets, lengths, prefix, mask: int32, on the device.  slopes
 * and table: fp32, on the device, finite and at most 1e20 and 1e30 in magnitude.  A table
 * may also hold -infinity (the pair is not seen) and lower finite values, the type's
 * lowest say, which count as some value below -1e30.  head_dim is a multiple of 8 up to
 * BBH_ATTEND_MAX_DIM; heads at most 65536, q_len * heads 2^30;
 * addresses of q, k, v and out are multiples of 16 bytes, their strides of 8 elements, row
 * strides below 2^23.  out and scratch overlap nothing.
 *
 * scratch (optional, 16-byte aligned): with it, calls with few rows spread the keys over
 * more workgroups and join their results; bbh_attend_scratch gives the bytes that it
 * pays to have (0: none), less is used as far as it goes.  Calls that overlap in time must
 * not share it.  Results differ in their last bits with the number of rows and the
 * scratch. */
#define BBH_ATTEND_MAX_DIM 256
typedef struct bbh_attend_args {
  bbh_heads q, k, v, out;
  int64_t q_rows, k_rows; /* packed: rows that exist */
  const int32_t *q_offsets, *k_offsets; /* (batch + 1) or NULL: padded */
  const int32_t *q_lengths, *k_lengths; /* (batch) or NULL */
  const int32_t *prefix;                /* (batch) or NULL */
  const int32_t *mask;                  /* (batch, k_len) or NULL */
  const float *slopes;                  /* (heads) or NULL */
  const float *table;                   /* (heads, 2 * table_half + 1) or NULL */
  void *scratch;
  size_t scratch_bytes;
  int batch, q_len, k_len; /* of the longest sequence */
  int heads, kv_heads, head_dim;
  int left, right, table_half;
  float scale, cap; /* between 2^-24 and 2^24; cap 0: none */
} bbh_attend_args;
bbh_status bbh_attend(const bbh_attend_args *args, bbh_stream_t stream);
/* Bytes of scratch for these sizes (pointers of args are not read, but those that are
 * NULL must be so in the call).  0 also for sizes that bbh_attend refuses. */
size_t bbh_attend_scratch(const bbh_attend_args *args);

#ifdef __cplusplus
}
#endif

#endif /* BBH_ATTEND_H */

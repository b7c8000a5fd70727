// bert_by_hand_attend.hpp - rotary positions and attention for models other than
// MiniLM (include/bbh_attend.h) in the C++ layer's manner: default arguments, an
// optional trailing stream, and errors that print and abort.  No counterpart in
// the reference.
#pragma once

#include <cmath>
#include <utility>

#include "bbh_attend.h"
#include "bert_by_hand.hpp"

// Heads that lie side by side in rows of `row` values (0: rows of nothing else), in
// sequences of `batch` values (padded ones; 0: packed rows).
inline bbh_heads heads_of(const __half *data, int heads, int head_dim, int64_t row = 0,
                          int64_t batch = 0) {
  bbh_heads t{};
  t.data = const_cast<__half *>(data);
  t.batch = batch;
  t.row = row ? row : (int64_t)heads * head_dim;
  t.head = head_dim;
  return t;
}

// A bbh_rope handle of its own.
class Rope {
 public:
  explicit Rope(const bbh_rope_config &config) { BBH_CHECK(bbh_rope_create(&config, &rope_)); }
  // The first rot_dim values of a head, unscaled.
  explicit Rope(int rot_dim, double base = 10000.0, bool interleaved = false)
      : Rope(plain(rot_dim, base, interleaved)) {}
  Rope(const Rope &) = delete;
  Rope &operator=(const Rope &) = delete;
  Rope(Rope &&o) noexcept : rope_(std::exchange(o.rope_, nullptr)) {}
  Rope &operator=(Rope &&o) noexcept {
    std::swap(rope_, o.rope_);
    return *this;
  }
  ~Rope() { bbh_rope_free(rope_); }
  const bbh_rope *get() const { return rope_; }

  // A configuration to fill in.
  static bbh_rope_config plain(int rot_dim, double base = 10000.0, bool interleaved = false) {
    bbh_rope_config c{};
    c.rot_dim = rot_dim;
    c.interleaved = interleaved ? 1 : 0;
    c.scaling = BBH_ROPE_NONE;
    c.base = base;
    c.magnitude = 1.0;
    return c;
  }

 private:
  bbh_rope *rope_ = nullptr;
};

// Arguments of launch_rope for q in place, every token at row % seq; k, v, positions, gammas
// and cache slots are filled in by the caller.
inline bbh_rope_args rope_args(bbh_heads q, int rows, int heads, int head_dim, int seq) {
  bbh_rope_args a{};
  a.q = a.q_out = q;
  a.rows = rows;
  a.seq = seq;
  a.heads = heads;
  a.head_dim = head_dim;
  a.eps = 1e-6f;
  return a;
}

// q and k normed and rotated, v moved (bbh_rope_heads); not with a Rope that was moved from.
inline void launch_rope(const Rope &rope, const bbh_rope_args &args, hipStream_t stream = nullptr) {
  BBH_CHECK(rope.get() ? bbh_rope_heads(rope.get(), &args, stream) : BBH_ERR_INVALID_ARG);
}

// The norms and the move alone.
inline void launch_head_norms(const bbh_rope_args &args, hipStream_t stream = nullptr) {
  BBH_CHECK(bbh_rope_heads(nullptr, &args, stream));
}

// Arguments of launch_attend for padded sequences: no window, cap, mask or bias, scores scaled by
// 1 / sqrt(head_dim).  The strides of q, k, v and out between sequences, where 0, become those
// of q_len and k_len rows.
inline bbh_attend_args attend_args(bbh_heads q, bbh_heads k, bbh_heads v, bbh_heads out, int batch,
                                   int q_len, int k_len, int heads, int kv_heads, int head_dim) {
  bbh_attend_args a{};
  auto placed = [](bbh_heads t, int len) {
    if (t.batch == 0) t.batch = t.row * len;
    return t;
  };
  a.q = placed(q, q_len);
  a.k = placed(k, k_len);
  a.v = placed(v, k_len);
  a.out = placed(out, q_len);
  a.batch = batch;
  a.q_len = q_len;
  a.k_len = k_len;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.left = a.right = -1;
  a.scale = 1.0f / std::sqrt((float)head_dim);
  return a;
}

// Attention (bbh_attend).
inline void launch_attend(const bbh_attend_args &args, hipStream_t stream = nullptr) {
  BBH_CHECK(bbh_attend(&args, stream));
}

// C ABI of rotary positions and of attention for models other than MiniLM
// (include/bbh_attend.h): argument validation, the rope handle.

#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <new>
#include <string>

#include "../../include/bbh_attend.h"
#include "attend.h"

using bbh::f16;

namespace bbh_detail {
bbh_status set_error(bbh_status s, const std::string& msg);  // capi.hip
}

struct bbh_rope {
  bbh::RopeSteps steps;
  int rot;
  bool interleaved;
  float magnitude;
  double freq[bbh::kMaxRopePairs];
};

namespace {

bbh_status fail(bbh_status s, const char* what, const char* msg) {
  return bbh_detail::set_error(s, std::string(what) + ": " + msg);
}
bbh_status invalid(const char* what, const char* msg) { return fail(BBH_ERR_INVALID_ARG, what, msg); }

bbh_status done(hipError_t e, const char* what) {
  if (e == hipSuccess) return BBH_OK;
  return bbh_detail::set_error(BBH_ERR_HIP, std::string(what) + ": " + hipGetErrorName(e) + " (" +
                                                hipGetErrorString(e) + ")");
}

bool off(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; }

// Largest stride and number of rows for which no element's offset leaves int64.
constexpr int64_t kMaxStride = (int64_t)1 << 40;
constexpr int kMaxLen = 1 << 28;

// A tensor of heads as memory: `batch` times `rows` rows of `heads` heads of dim fp16 values.
struct Region {
  const void* data;
  int64_t batch, batch_stride, rows, row, heads, head, dim;
  bool none() const { return !data || batch < 1 || rows < 1 || heads < 1; }
  uintptr_t begin() const { return (uintptr_t)data; }
  // (as far as addresses go: sizes that no memory holds overlap what lies behind them)
  uintptr_t end() const {
    const __int128 e = (__int128)begin() + 2 * ((__int128)(batch - 1) * batch_stride +
                                                (__int128)(rows - 1) * row + (heads - 1) * head + dim);
    return e > (__int128)UINTPTR_MAX ? UINTPTR_MAX : (uintptr_t)e;
  }
  int64_t width() const { return (heads - 1) * head + dim; }  // of a row
};

// Whether two regions share memory, taking it as read that they do where that is not plain:
// apart in memory, or columns of the same rows, or of the same heads of them (q, k and v of a head
// side by side).
bool overlap(const Region& a, const Region& b) {
  if (a.none() || b.none()) return false;
  if (a.begin() >= b.end() || b.begin() >= a.end()) return false;
  const int64_t row = a.row;
  const bool same_rows = row == b.row && row > 0 && a.width() <= row && b.width() <= row &&
                         (a.batch == 1 || a.batch_stride % row == 0) &&
                         (b.batch == 1 || b.batch_stride % row == 0);
  if (!same_rows) return true;
  const int64_t bytes = (int64_t)(b.begin() - a.begin());
  if (bytes % 2) return true;
  int64_t d = bytes / 2 % row;  // b's first column, seen from a's
  if (d < 0) d += row;
  const bool wraps = d + b.width() > row;  // b's last columns lie in a's next row
  if (d >= a.width() && !wraps) return false;
  const int64_t head = a.heads > 1 ? a.head : b.head;
  if (head < 1 || (b.heads > 1 && b.head != head) || (wraps && row % head)) return true;
  return !(d % head >= a.dim && d % head + b.dim <= head);
}

// Whether an output's elements are apart from each other.
bool apart(const Region& r) {
  if (r.none()) return true;
  if (r.heads > 1 && r.head < r.dim) return false;
  if (r.rows > 1 && r.row < r.dim) return false;
  const __int128 column = (__int128)(r.rows - 1) * r.row + r.dim;
  if (r.rows > 1 && r.heads > 1) {
    // rows of heads, or heads of rows
    if (r.row < r.width() && r.head < column) return false;
  }
  if (r.batch > 1) {
    const __int128 one = column + (r.heads - 1) * r.head;
    if (r.batch_stride < one &&
        !(r.row > 0 && r.width() <= r.batch_stride &&
          r.row >= (__int128)(r.batch - 1) * r.batch_stride + r.width()))
      return false;
  }
  return true;
}

bool strides_ok(const bbh_heads& t) {
  return t.row >= 0 && t.head >= 0 && t.batch >= 0 && t.row <= kMaxStride && t.head <= kMaxStride &&
         t.batch <= kMaxStride;
}

}  // namespace

static_assert(BBH_ROPE_MAX_DIM == 2 * bbh::kMaxRopePairs, "limits");

extern "C" {

bbh_status bbh_rope_create(const bbh_rope_config* c, bbh_rope** out) {
  const char* what = "bbh_rope_create";
  if (!out) return invalid(what, "null argument");
  *out = nullptr;
  if (!c) return invalid(what, "null argument");
  if (c->rot_dim < 2 || c->rot_dim % 2)
    return invalid(what, "rot_dim must be even and positive");
  if (c->rot_dim > BBH_ROPE_MAX_DIM)
    return fail(BBH_ERR_UNSUPPORTED, what, "rot_dim above 256 is not supported");
  if (!isfinite((float)c->magnitude)) return invalid(what, "magnitude must be finite in fp32");
  const int pairs = c->rot_dim / 2;
  double f[bbh::kMaxRopePairs];
  if (c->frequencies) {
    for (int i = 0; i < pairs; ++i) f[i] = c->frequencies[i];
  } else {
    if (!(c->base > 1) || !isfinite(c->base)) return invalid(what, "base must be finite and above 1");
    if (c->scaling < BBH_ROPE_NONE || c->scaling > BBH_ROPE_BANDS)
      return invalid(what, "unknown scaling");
    if (c->scaling != BBH_ROPE_NONE && (!(c->factor >= 1) || !isfinite(c->factor)))
      return invalid(what, "factor must be finite and at least 1");
    const bool turns = c->scaling == BBH_ROPE_RAMP || c->scaling == BBH_ROPE_BANDS;
    if (turns && (!(c->original > 0) || !isfinite(c->original)))
      return invalid(what, "original must be finite and positive");
    if (turns && (!(c->low > 0) || !(c->high > c->low) || !isfinite(c->high)))
      return invalid(what, "low and high must be finite, 0 < low < high");
    const double rot = c->rot_dim, two_pi = 2 * M_PI;
    double base = c->base;
    if (c->scaling == BBH_ROPE_BASE && c->rot_dim > 2) base *= pow(c->factor, rot / (rot - 2));
    double first = 0, last = 0;
    if (c->scaling == BBH_ROPE_RAMP) {
      auto pair = [&](double n) { return rot * log(c->original / (two_pi * n)) / (2 * log(base)); };
      first = fmin(fmax(floor(pair(c->high)), 0), rot - 1);
      last = fmin(fmax(ceil(pair(c->low)), 0), rot - 1);
    }
    for (int i = 0; i < pairs; ++i) {
      const double g = pow(base, -2.0 * i / rot);
      f[i] = g;
      if (c->scaling == BBH_ROPE_LINEAR) f[i] = g / c->factor;
      if (c->scaling == BBH_ROPE_RAMP) {
        const double r = fmin(fmax((i - first) / fmax(last - first, 0.001), 0), 1);
        f[i] = g * (1 - r) + g / c->factor * r;
      }
      if (c->scaling == BBH_ROPE_BANDS) {
        const double t = (c->original * g / two_pi - c->low) / (c->high - c->low);
        const double s = fmin(fmax(t, 0), 1);
        f[i] = g * s + g / c->factor * (1 - s);
      }
    }
  }
  for (int i = 0; i < pairs; ++i)
    if (!isfinite(f[i])) return invalid(what, "frequencies must be finite");
  bbh_rope* r = new (std::nothrow) bbh_rope();
  if (!r) return fail(BBH_ERR_OOM, what, "no host memory");
  r->rot = c->rot_dim;
  r->interleaved = c->interleaved != 0;
  r->magnitude = (float)c->magnitude;
  for (int i = 0; i < pairs; ++i) {
    r->freq[i] = f[i];
    // turns a position, of which whole ones do not matter, in units of 2^-64
    const long double t = (long double)f[i] / 6.283185307179586476925286766559L;
    const long double frac = t - floorl(t);  // [0, 1)
    const long double units = roundl(ldexpl(frac, 64));
    const uint64_t n = units >= 18446744073709551616.0L ? 0 : (uint64_t)units;
    r->steps.step[i] = make_uint2((uint32_t)n, (uint32_t)(n >> 32));
  }
  *out = r;
  return BBH_OK;
}

bbh_status bbh_rope_free(bbh_rope* rope) {
  delete rope;
  return BBH_OK;
}

bbh_status bbh_rope_frequencies(const bbh_rope* rope, double* out) {
  if (!rope || !out) return invalid("bbh_rope_frequencies", "null argument");
  memcpy(out, rope->freq, sizeof(double) * (rope->rot / 2));
  return BBH_OK;
}

bbh_status bbh_rope_heads(const bbh_rope* rope, const bbh_rope_args* a, bbh_stream_t stream) {
  const char* what = "bbh_rope_heads";
  if (!a || !a->q.data || !a->q_out.data) return invalid(what, "null argument");
  const bool k = a->k.data != nullptr, v = a->v.data != nullptr;
  if (k != (a->k_out.data != nullptr) || v != (a->v_out.data != nullptr))
    return invalid(what, "k and k_out, v and v_out go together");
  if (a->rows < 0) return invalid(what, "rows must not be negative");
  if (a->heads < 1 || ((k || v) && a->kv_heads < 1) || a->head_dim < 1)
    return invalid(what, "heads and head_dim must be positive");
  if (a->head_dim > BBH_ROPE_MAX_DIM)
    return fail(BBH_ERR_UNSUPPORTED, what, "heads longer than 256 are not supported");
  if (a->heads > 65536 || a->kv_heads > 65536)
    return fail(BBH_ERR_UNSUPPORTED, what, "more than 65536 heads are not supported");
  if (rope && rope->rot > a->head_dim) return invalid(what, "rot_dim exceeds head_dim");
  if (rope && !a->positions && a->seq < 1) return invalid(what, "seq must be positive without positions");
  const bool norm = a->q_gamma || a->k_gamma;
  if (norm && (!(a->eps >= 0.f) || !isfinite(a->eps)))
    return invalid(what, "eps must be finite and not negative");
  if (a->k_gamma && !k) return invalid(what, "k_gamma without k");
  if (a->kv_rows && !k && !v) return invalid(what, "kv_rows without k or v");
  if (a->kv_rows && (a->kv_out_rows < 0 || a->kv_out_rows > kMaxStride))
    return invalid(what, "kv_out_rows out of range");
  const bbh_heads* all[6] = {&a->q, &a->k, &a->v, &a->q_out, &a->k_out, &a->v_out};
  for (const bbh_heads* t : all) {
    if (!t->data) continue;
    if (!strides_ok(*t)) return invalid(what, "strides must not be negative (or above 2^40)");
    if (off(t->data, 2)) return invalid(what, "fp16 operands must be 2-byte aligned");
  }
  if (off(a->q_gamma, 2) || off(a->k_gamma, 2)) return invalid(what, "fp16 operands must be 2-byte aligned");
  if (off(a->positions, 4) || off(a->kv_rows, 8))
    return invalid(what, "positions must be 4-byte and kv_rows 8-byte aligned");
  auto region = [&](const bbh_heads& t, int heads, int64_t rows) {
    return Region{t.data, 1, 0, rows, t.row, heads, t.head, a->head_dim};
  };
  const int64_t kv_rows = a->kv_rows ? a->kv_out_rows : a->rows;
  Region in[3] = {region(a->q, a->heads, a->rows), region(a->k, a->kv_heads, a->rows),
                  region(a->v, a->kv_heads, a->rows)};
  Region out[3] = {region(a->q_out, a->heads, a->rows), region(a->k_out, a->kv_heads, kv_rows),
                   region(a->v_out, a->kv_heads, kv_rows)};
  for (int i = 0; i < 3; ++i) {
    if (!apart(out[i])) return invalid(what, "an output's rows or heads overlap");
    for (int j = 0; j < 3; ++j) {
      if (i < j && overlap(out[i], out[j])) return invalid(what, "outputs overlap");
      const bool in_place = i == j && out[i].data == in[j].data && out[i].row == in[j].row &&
                            out[i].head == in[j].head && (i == 0 || !a->kv_rows);
      if (!in_place && overlap(out[i], in[j])) return invalid(what, "an output overlaps an input");
    }
    const Region small[4] = {
        {a->q_gamma, 1, 0, 1, 0, 1, 0, a->head_dim},
        {a->k_gamma, 1, 0, 1, 0, 1, 0, a->head_dim},
        {a->positions, 1, 0, 1, 0, 1, 0, 2 * (int64_t)a->rows},
        {a->kv_rows, 1, 0, 1, 0, 1, 0, 4 * (int64_t)a->rows}};
    for (const Region& r : small)
      if (a->rows > 0 && overlap(out[i], r)) return invalid(what, "an output overlaps an input");
  }
  if (a->rows == 0) return BBH_OK;
  bbh::RopeParams p{};
  auto part = [](const bbh_heads& x, const bbh_heads& y, const void* gamma, int heads) {
    return bbh::RopeParams::Part{static_cast<const f16*>(x.data), static_cast<f16*>(y.data),
                                 static_cast<const f16*>(gamma), x.row, x.head, y.row, y.head, heads};
  };
  p.q = part(a->q, a->q_out, a->q_gamma, a->heads);
  p.k = part(a->k, a->k_out, a->k_gamma, k ? a->kv_heads : 0);
  p.v = part(a->v, a->v_out, nullptr, v ? a->kv_heads : 0);
  p.positions = a->positions;
  p.kv_rows = a->kv_rows;
  p.kv_out_rows = a->kv_out_rows;
  p.rows = a->rows;
  p.seq = a->seq;
  p.dim = a->head_dim;
  p.rot = rope ? rope->rot : 0;
  p.interleaved = rope && rope->interleaved;
  p.eps = a->eps;
  p.magnitude = rope ? rope->magnitude : 1.f;
  static const bbh::RopeSteps no_steps{};
  return done(bbh::rope_heads(p, rope ? rope->steps : no_steps, static_cast<hipStream_t>(stream)), what);
}

static bbh_status attend_params(const bbh_attend_args* a, bbh::AttendParams& p) {
  const char* what = "bbh_attend";
  if (a->batch < 0 || a->q_len < 0 || a->k_len < 0)
    return invalid(what, "batch, q_len and k_len must not be negative");
  if (a->heads < 1 || a->kv_heads < 1 || a->head_dim < 1)
    return invalid(what, "heads, kv_heads and head_dim must be positive");
  if (a->heads % a->kv_heads) return invalid(what, "heads must be a multiple of kv_heads");
  if (a->head_dim % 8 || a->head_dim > BBH_ATTEND_MAX_DIM)
    return fail(BBH_ERR_UNSUPPORTED, what, "head_dim must be a multiple of 8 up to 256");
  const int group = a->heads / a->kv_heads;
  if (a->q_len > kMaxLen || a->k_len > kMaxLen || (int64_t)a->q_len * group > kMaxLen)
    return fail(BBH_ERR_UNSUPPORTED, what, "k_len or q_len * heads / kv_heads above 2^28");
  if ((int64_t)a->batch * a->heads > INT_MAX)
    return fail(BBH_ERR_UNSUPPORTED, what, "batch * heads above 2^31 - 1");
  // (a sequence's work-items fit a launch's 2^32)
  if (a->heads > 65536 || (int64_t)a->q_len * a->heads > 1 << 30)
    return fail(BBH_ERR_UNSUPPORTED, what, "more than 65536 heads, or q_len * heads above 2^30");
  // (so that biases divided by either keep their size)
  constexpr float kLeast = 0x1p-24f, kMost = 0x1p24f;
  if (!(a->scale >= kLeast && a->scale <= kMost))
    return invalid(what, "scale must lie between 2^-24 and 2^24");
  if (!(a->cap == 0.f || (a->cap >= kLeast && a->cap <= kMost)))
    return invalid(what, "cap must be 0 or lie between 2^-24 and 2^24");
  if (a->table && (a->table_half < 0 || a->table_half > kMaxLen))
    return invalid(what, "table_half out of range");
  if ((a->q_offsets && a->q_rows < 0) || (a->k_offsets && a->k_rows < 0))
    return invalid(what, "rows must not be negative");
  auto heads = [](const bbh_heads& t) { return bbh::Heads{t.batch, t.row, t.head}; };
  p.q = static_cast<const f16*>(a->q.data);
  p.k = static_cast<const f16*>(a->k.data);
  p.v = static_cast<const f16*>(a->v.data);
  p.out = static_cast<f16*>(a->out.data);
  p.qs = heads(a->q);
  p.ks = heads(a->k);
  p.vs = heads(a->v);
  p.os = heads(a->out);
  // (a row that is the only one has no stride that matters, and rows behind it have to be elsewhere)
  if ((a->k_offsets ? a->k_rows : a->k_len) <= 1) p.ks.row = p.vs.row = a->head_dim;
  p.q_offsets = a->q_offsets;
  p.k_offsets = a->k_offsets;
  p.q_lengths = a->q_lengths;
  p.k_lengths = a->k_lengths;
  p.prefix = a->prefix;
  p.mask = a->mask;
  p.slopes = a->slopes;
  p.table = a->table;
  p.q_rows = a->q_rows;
  p.k_rows = a->k_rows;
  p.batch = a->batch;
  p.q_len = a->q_len;
  p.k_len = a->k_len;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.dim = a->head_dim;
  p.group = group;
  // no bound is further than the longest sequences reach
  p.left = a->left < 0 || a->left > 2 * kMaxLen ? -1 : a->left;
  p.right = a->right < 0 || a->right > 2 * kMaxLen ? -1 : a->right;
  p.half = a->table_half;
  const double log2e = 1.4426950408889634;
  const bool near = a->cap > 0.f && a->cap <= bbh::kNearCap, wide = a->cap > bbh::kNearCap;
  const double unit = near ? 2.0 * a->cap : wide ? a->cap : a->scale;
  p.mscale = (float)(unit * log2e);
  p.bias_scale = (float)(1.0 / unit);
  p.cap_k = near ? (float)(2 * log2e * a->scale / a->cap) : wide ? a->scale / a->cap : 0.f;
  p.wide_cap = wide;
  return BBH_OK;
}

bbh_status bbh_attend(const bbh_attend_args* a, bbh_stream_t stream) {
  const char* what = "bbh_attend";
  if (!a) return invalid(what, "null argument");
  bbh::AttendParams p{};
  const bbh_status st = attend_params(a, p);
  if (st != BBH_OK) return st;
  if (a->batch == 0 || a->q_len == 0) return BBH_OK;
  const bool no_keys = a->k_len == 0 || (a->k_offsets && a->k_rows == 0);
  if (!a->q.data || !a->out.data || (!no_keys && (!a->k.data || !a->v.data)))
    return invalid(what, "null argument");
  for (const bbh_heads* t : {&a->q, &a->k, &a->v, &a->out}) {
    if (off(t->data, 16)) return invalid(what, "q, k, v and out must be 16-byte aligned");
    if (!strides_ok(*t)) return invalid(what, "strides must not be negative (or above 2^40)");
    if ((t->batch | t->row | t->head) & 7) return invalid(what, "strides must be multiples of 8");
    if (t->row >= (1 << 23)) return fail(BBH_ERR_UNSUPPORTED, what, "row strides of 2^23 or more");
  }
  for (const void* t : {(const void*)a->q_offsets, (const void*)a->k_offsets, (const void*)a->q_lengths,
                        (const void*)a->k_lengths, (const void*)a->prefix, (const void*)a->mask,
                        (const void*)a->slopes, (const void*)a->table})
    if (off(t, 4)) return invalid(what, "int32 and fp32 operands must be 4-byte aligned");
  if (a->scratch && off(a->scratch, 16)) return invalid(what, "scratch must be 16-byte aligned");
  auto region = [&](const bbh_heads& t, bool packed, int64_t rows, int len, int heads) {
    return packed ? Region{t.data, 1, 0, rows, t.row, heads, t.head, a->head_dim}
                  : Region{t.data, a->batch, t.batch, len, t.row, heads, t.head, a->head_dim};
  };
  const Region out = region(a->out, a->q_offsets, a->q_rows, a->q_len, a->heads);
  const Region in[3] = {region(a->q, a->q_offsets, a->q_rows, a->q_len, a->heads),
                        region(a->k, a->k_offsets, a->k_rows, a->k_len, a->kv_heads),
                        region(a->v, a->k_offsets, a->k_rows, a->k_len, a->kv_heads)};
  if (!apart(out)) return invalid(what, "rows or heads of out overlap");
  for (const Region& r : in)
    if (overlap(out, r)) return invalid(what, "out overlaps an input");
  auto words = [](const void* data, int64_t n) { return Region{data, 1, 0, 1, 0, 1, 0, 2 * n}; };
  const Region small[8] = {
      words(a->q_offsets, (int64_t)a->batch + 1), words(a->k_offsets, (int64_t)a->batch + 1),
      words(a->q_lengths, a->batch),              words(a->k_lengths, a->batch),
      words(a->prefix, a->batch),                 words(a->mask, (int64_t)a->batch * a->k_len),
      words(a->slopes, a->heads),                 words(a->table, a->heads * (2 * (int64_t)a->table_half + 1))};
  const Region sc{a->scratch, 1, 0, 1, 0, 1, 0, (int64_t)(a->scratch_bytes / 2)};
  for (const Region& r : small) {
    if (overlap(out, r)) return invalid(what, "out overlaps an input");
    if (overlap(sc, r)) return invalid(what, "scratch overlaps an operand");
  }
  if (overlap(sc, out) || overlap(sc, in[0]) || overlap(sc, in[1]) || overlap(sc, in[2]))
    return invalid(what, "scratch overlaps an operand");
  return done(bbh::attend(p, a->scratch, a->scratch ? a->scratch_bytes : 0,
                          static_cast<hipStream_t>(stream)),
              what);
}

size_t bbh_attend_scratch(const bbh_attend_args* a) {
  bbh::AttendParams p{};
  if (!a || attend_params(a, p) != BBH_OK || a->batch == 0 || a->q_len == 0) return 0;
  return bbh::attend_scratch(p);
}

}  // extern "C"

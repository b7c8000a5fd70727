"""Attention for other models (include/bbh_attend.h): scores far from zero and under
large caps, small weights, every tile of a long cache, scratch of any size.

u is half a step of fp32 relative to the value, 2^-24; H the same of fp16,
2^-11; below fp16's normal range a rounding is off by up to 2^-25."""

import math

import pytest

from test_attend import H, TINY, U, _gen, _normal

gpu = pytest.mark.gpu


# Scores of caps up to this are computed from an exponential next to 1, to half a
# step of fp32 of the cap; those of larger ones to a few steps of their own size.
NEAR_CAP = 128.0


def _attend64(torch, q, k, v, right=-1, scale=None, cap=0.0, slopes=None, table=None):
    """One sequence in 64 bits, and what a result may be off by, where only scores that
    carry weight count: a key of weight 0 may have a score of any size."""
    q, k, v = q.double(), k.double(), v.double()
    (nq, h, d), nk = q.shape, k.shape[0]
    rep = h // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    scale = d ** -0.5 if scale is None else scale
    qt, kt = q.transpose(0, 1), k.permute(1, 2, 0).contiguous()
    s = torch.matmul(qt, kt) * scale
    off = torch.matmul(qt.abs(), kt.abs()) * scale * (d + 4) * U  # fp32 sums of D products
    if cap:
        s = cap * torch.tanh(s / cap)
        # the small ones: twice the cap times 1 / (1 + e), whose exponential (a quarter of 2 u),
        # sum (u) and reciprocal (2 u) are off by less than 4 u together; the large ones: the
        # argument (2 u) and a quotient of polynomials (6 u), or, of a result above 0.6, the
        # same four and a difference
        off = off + (8 * min(cap, NEAR_CAP) + 16 * s.abs()) * U
    dist = torch.arange(nk, device="cuda") - (torch.arange(nq, device="cuda")[:, None] + nk - nq)
    for b in ([] if slopes is None else [-slopes.double()[:, None, None] * dist.abs()]) + \
            ([] if table is None else
             [table.double()[:, dist.clamp(-(table.shape[1] // 2), table.shape[1] // 2) + table.shape[1] // 2]]):
        s, off = s + b, off + 3 * U * (b.abs() + s.abs())
    if right >= 0:
        s = s.masked_fill(dist > right, -math.inf)
    p = torch.softmax(s, -1)
    # difference from the maximum and its product, rounded each
    carry = p > 1e-12
    off = torch.where(carry, off + 4 * U * s.abs(), 0.0).amax(-1, keepdim=True)
    v = v.transpose(0, 1).contiguous()
    out, size = torch.matmul(p, v), torch.matmul(p, v.abs())
    # weights rounded to fp16 (those below 2^-21 of the largest by up to 2^-32 of it);
    # the output rounded once; fp32 sums
    small = torch.matmul(((p > 0) & (p < 2 ** -13)).double(), v.abs()) * 2.0 ** -32
    tol = H * out.abs() + size * (2 * H + 4 * off + 2 * (nk ** 0.5 + 40) * U) + small + TINY + 1e-12 * nk
    return out.transpose(0, 1), tol.transpose(0, 1)


def _worst(torch, got, want, tol):
    ratio = (got.double() - want).abs() / tol
    assert bool(ratio.isfinite().all())
    return float(ratio.max())


# a set of kernels each: q_len, k_len, heads, kv_heads
SETS = [(9, 9, 2, 2), (1, 500, 4, 2), (60, 60, 2, 2), (300, 300, 4, 2), (1100, 1100, 1, 1), (2, 66000, 4, 4)]


@gpu
@pytest.mark.parametrize("cap", [128.0, 129.0, 1e3, 1e5, 2.0 ** 24])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("q_len,k_len,heads,kv", SETS)
def test_caps_of_any_size(torch_cuda, q_len, k_len, heads, kv, dim, cap):
    """Ordinary scores, ones of the cap's size, and biases beside them."""
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, k_len + dim)
    q = _normal(torch, g, 1, q_len, heads, dim)
    k, v = _normal(torch, g, 1, k_len, kv, dim), _normal(torch, g, 1, k_len, kv, dim)
    slopes = 0.05 * torch.rand(heads, device="cuda", generator=g)
    table = torch.randn(heads, 41, device="cuda", generator=g)
    scratch = torch.empty(1 << 22, device="cuda")
    for kw in (dict(), dict(scale=3 * dim ** -0.5), dict(slopes=slopes), dict(table=table, right=0),
               dict(scale=min(0.5 * cap * dim ** -0.5, 200.0))):
        out = torch.full_like(q, float("nan"))
        engine.launch_attend(q, k, v, out, cap=cap, scratch=scratch, **kw)
        torch.cuda.synchronize()
        want, tol = _attend64(torch, q[0], k[0], v[0], cap=cap, **kw)
        assert _worst(torch, out[0], want, tol) <= 1, kw.keys()


@gpu
@pytest.mark.parametrize("far", [-3e4, -1e6, -1e9, -3.4e38])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_len,k_len,heads,kv", SETS[1:])
def test_a_table_that_hides_by_large_values(torch_cuda, q_len, k_len, heads, kv, dim, far):
    """The first keys of a row far below the ones behind them, as masks of -1e9 have it: the
    latter's weights are those of their own differences."""
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, k_len + dim)
    q = _normal(torch, g, 1, q_len, heads, dim)
    k, v = _normal(torch, g, 1, k_len, kv, dim), _normal(torch, g, 1, k_len, kv, dim)
    table = torch.randn(heads, 401, device="cuda", generator=g)
    table[:, :180] = far  # more than 20 keys back
    table[:, 230:] = far  # 30 and more ahead
    scratch = torch.empty(1 << 22, device="cuda")
    for cap in (0.0, 30.0):
        for sc in (None, scratch):
            out = torch.full_like(q, float("nan"))
            engine.launch_attend(q, k, v, out, table=table, cap=cap, scratch=sc)
            torch.cuda.synchronize()
            want, tol = _attend64(torch, q[0], k[0], v[0], table=table, cap=cap)
            assert _worst(torch, out[0], want, tol) <= 1, (cap, sc is None)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len", [1, 64])
@pytest.mark.parametrize("nk", [3000, 100000])
def test_steep_slopes_over_a_long_cache(torch_cuda, nk, q_len, dim):
    """In one pass and split: the first keys' scores lie as far as -2e6, those that carry weight
    near zero."""
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, nk + dim)
    q = 3 * _normal(torch, g, 1, q_len, 6, dim)
    k, v = _normal(torch, g, 1, nk, 6, dim), _normal(torch, g, 1, nk, 6, dim)
    slopes = torch.tensor([0.4, 0.6, 0.84, 1.0, 3.0, 20.0], device="cuda")
    for sc in (None, torch.empty(1 << 22, device="cuda")):
        out = torch.full_like(q, float("nan"))
        engine.launch_attend(q, k, v, out, right=0, slopes=slopes, scratch=sc)
        torch.cuda.synchronize()
        # (keys further back than this weigh less than e^-700 against the query's own)
        n = min(nk, 3000 + q_len)
        want, tol = _attend64(torch, q[0], k[0, -n:], v[0, -n:], right=0, slopes=slopes)
        assert _worst(torch, out[0], want, tol) <= 1, sc is None


@gpu
@pytest.mark.parametrize("gap", [15.5, 17.25, 18.0, 19.0])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_len,scratch", [(1, False), (1, True), (33, False), (700, False)])
def test_a_long_flat_tail_keeps_its_values(torch_cuda, q_len, scratch, dim, gap):
    """One key `gap` above 131071 equal ones, whose values alone are not zero: each weighs less
    than 2^-22 of it, all of them 2e-2 to 7e-4."""
    from bbh import engine

    torch = torch_cuda
    n = 131072
    q = torch.zeros(1, q_len, 1, dim, device="cuda").half()
    k, v = torch.zeros(1, n, 1, dim, device="cuda").half(), torch.ones(1, n, 1, dim, device="cuda").half()
    q[..., 3], k[0, 0, 0, 3], v[0, 0] = 1.0, gap, 0.0
    out = torch.full_like(q, float("nan"))
    engine.launch_attend(q, k, v, out, scale=1.0,
                         scratch=torch.empty(1 << 22, device="cuda") if scratch else None)
    torch.cuda.synchronize()
    tail = (n - 1) * math.exp(-gap)
    want = tail / (1 + tail)
    # each weight is off by up to 2^-32 of the largest; sums of up to 4096 tiles in fp32, the
    # output rounded
    tol = want * (2 * H + 2 * 8192 * U) + n * 2.0 ** -32 + TINY
    assert float((out.double() - want).abs().max()) <= tol, float(out.double().mean() / want)


# batch, q_len, k_len, heads a key/value head, with scratch: kernels of a wavefront or four over
# tiles in turn, of rows, split and not
CACHES = [(1, 1, 70001, 2, True), (1, 1, 70001, 2, False), (1, 5, 70001, 1, True), (1, 1, 4003, 1, True),
          (1, 3, 4003, 2, False), (70, 1, 1000, 1, True), (70, 1, 1000, 1, False), (1, 40, 9000, 1, True),
          (1, 40, 9000, 1, False), (1, 300, 9000, 1, True), (3, 17, 140, 1, False)]


@gpu
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("form", ["plain", "cap", "any", "window", "behind"])
@pytest.mark.parametrize("batch,q_len,nk,group,scratch", CACHES)
def test_every_tile_of_a_cache_counts_once(torch_cuda, batch, q_len, nk, group, scratch, form, dim):
    """Equal scores, and each value of each key/value head from 32 keys of its own: a tile (or a key
    of it) that is lost, read twice or weighed otherwise shows in the value of its own."""
    from bbh import engine

    torch = torch_cuda
    tiles = (nk + 31) // 32
    kv = (tiles + dim - 1) // dim
    if batch > 1:
        kv = max(kv, 16)
    j = torch.arange(nk, device="cuda")
    amount = 1 + j % 7
    v = torch.zeros(nk, kv * dim, device="cuda", dtype=torch.float16)
    v[j, j // 32] = amount.half()
    v = v.view(1, nk, kv, dim).expand(batch, -1, -1, -1)
    q = torch.zeros(batch, q_len, kv * group, dim, device="cuda").half()
    k = _normal(torch, _gen(torch, nk), 1, nk, kv, dim).expand(batch, -1, -1, -1)
    kw = {"plain": {}, "cap": dict(cap=8.0), "any": dict(slopes=torch.zeros(kv * group, device="cuda")),
          "window": dict(left=nk - 45, right=0, prefix=torch.full((batch,), 10, device="cuda", dtype=torch.int32),
                         mask=(j % 11 != 5).int().expand(batch, -1).contiguous()),
          "behind": dict(left=nk // 3)}[form]
    seen = torch.ones(q_len, nk, dtype=torch.bool, device="cuda")
    if form == "window":
        i = torch.arange(q_len, device="cuda")[:, None] + nk - q_len
        seen = ((j <= i) & (j >= i - (nk - 45)) | (j < 10)) & (j % 11 != 5)
    elif form == "behind":
        seen = j >= torch.arange(nk - q_len, nk, device="cuda")[:, None] - nk // 3
    each = torch.zeros(q_len, kv * dim, device="cuda", dtype=torch.float64)
    each.index_add_(1, j // 32, seen.double() * amount)
    want = (each / seen.sum(-1, keepdim=True)).view(q_len, kv, dim).repeat_interleave(group, 1)
    out = torch.full_like(q, float("nan"))
    room = torch.empty(max(engine.attend_scratch(q, k, v, out, **kw), 16), dtype=torch.uint8, device="cuda")
    engine.launch_attend(q, k, v, out, scratch=room if scratch else None, **kw)
    torch.cuda.synchronize()
    # weights of exactly one power of two (under a cap to some steps of it, all alike), sums of
    # whole numbers below 2^24: the reciprocal, the product and the output are rounded
    assert bool(((out.double() - want).abs() <= (H + 64 * U) * want + TINY).all())


@gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_len,nk,heads,kv", [(1, 300000, 4, 2), (5, 100003, 8, 4), (1, 40000, 12, 12)])
def test_scratch_too_small_to_split_is_as_none(torch_cuda, q_len, nk, heads, kv, dim):
    """Less scratch than it pays to have is used as far as it goes: none of it where it does not
    hold two parts, and the call is the one without."""
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, nk)
    q = _normal(torch, g, 1, q_len, heads, dim)
    k, v = _normal(torch, g, 1, nk, kv, dim), _normal(torch, g, 1, nk, kv, dim)
    whole = torch.empty_like(q)
    engine.launch_attend(q, k, v, whole)
    full = torch.empty_like(q)
    most = engine.attend_scratch(q, k, v, full)
    engine.launch_attend(q, k, v, full, scratch=torch.empty(most, dtype=torch.uint8, device="cuda"))
    part = q_len * heads * (4 * dim + 8)
    for n, same in ((16, True), (2 * part - 16, True), (2 * part, False), (3 * part, False), (most // 2, False)):
        out = torch.full_like(q, float("nan"))
        engine.launch_attend(q, k, v, out, scratch=torch.empty(n, dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        assert not same or torch.equal(out, whole), n
        # values of deviation (e / nk)^1/2 whose weights are rounded to fp16 at random on both
        # sides, less than H of that each (ten of them allowed), and both outputs' own roundings
        tol = 2 * H * full.double().abs() + 16 * H * nk ** -0.5 + 2 * TINY
        assert bool(((out.double() - full.double()).abs() <= tol).all()), n


@pytest.mark.parametrize("left,right", [(0, 0), (500, 0), (500, -1), (500, 7), (500, 1 << 28), (100000, -1)])
@pytest.mark.parametrize("q_len", [1, 3, 40, 3000])
def test_scratch_for_the_keys_that_a_window_leaves(q_len, left, right):
    """The queries stand at the last keys: a bound behind them, or none, adds no key to what
    their windows hold."""
    import ctypes

    from test_attend import _args, _lib

    def bytes_of(**kw):
        return _lib().bbh_attend_scratch(ctypes.byref(_args(batch=1, q_len=q_len, **kw)))

    seen = min(1000000, q_len + left)
    assert bytes_of(k_len=1000000, left=left, right=right) == bytes_of(k_len=seen, left=-1, right=-1)

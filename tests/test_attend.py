"""Rotary positions and attention for other models (include/bbh_attend.h):
refusals on the CPU, numerics on the GPU against the formulas in 64 bits.

u is half a step of fp32 relative to the value, 2^-24; H the same of fp16,
2^-11; below fp16's normal range a rounding is off by up to 2^-25."""

import ctypes
import math
import os
import re

import numpy as np
import pytest

from conftest import ROOT

U, H, TINY = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25
gpu = pytest.mark.gpu


# ---- CPU: declarations and refusals -------------------------------------------

def _lib():
    from bbh import capi

    return capi.lib()


def test_header_declarations_all_exported():
    from bbh import capi

    text = open(os.path.join(ROOT, "include", "bbh_attend.h")).read()
    names = sorted(set(re.findall(r"^(?:bbh_status|size_t) (bbh_[a-z0-9_]+)\s*\(", text, re.M)))
    assert len(names) == 6 and sorted(capi.SIGNATURES_ATTEND) == names
    for n in names:
        assert hasattr(_lib(), n), n


def test_structs_have_the_header_s_fields():
    from bbh import capi

    text = open(os.path.join(ROOT, "include", "bbh_attend.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for struct, cls in (("bbh_rope_config", capi.RopeConfig), ("bbh_rope_args", capi.RopeArgs),
                        ("bbh_attend_args", capi.AttendArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
        fields = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            kind, names = re.match(r"((?:const )?\w+)\s+(.*)", decl, re.S).groups()
            for n in names.split(","):
                n = n.strip().lstrip("*")
                fields += [f"{n}_{x}" for x in ("data", "batch", "row", "head")] \
                    if kind == "bbh_heads" else [n]
        assert [f[0] for f in cls._fields_] == fields, struct


P = 1 << 30  # fake operands, 1 GB apart; refusals come before any device work


def _rope_config(**change):
    from bbh import capi

    a = dict(rot_dim=64, interleaved=0, scaling=0, base=10000.0, factor=1.0, original=0.0, low=0.0,
             high=0.0, magnitude=1.0)
    a.update(change)
    return capi.RopeConfig(**a)


@pytest.mark.parametrize("change, status, message", [
    (dict(rot_dim=0), 1, b"rot_dim"), (dict(rot_dim=7), 1, b"rot_dim"), (dict(rot_dim=-2), 1, b"rot_dim"),
    (dict(rot_dim=258), 7, b"256"), (dict(base=1.0), 1, b"base"), (dict(base=math.nan), 1, b"base"),
    (dict(base=math.inf), 1, b"base"), (dict(scaling=5), 1, b"scaling"), (dict(scaling=-1), 1, b"scaling"),
    (dict(scaling=1, factor=0.5), 1, b"factor"), (dict(scaling=2, factor=math.nan), 1, b"factor"),
    (dict(scaling=3, factor=2.0, low=1.0, high=32.0), 1, b"original"),
    (dict(scaling=3, factor=2.0, original=4096.0), 1, b"low"),
    (dict(scaling=4, factor=2.0, original=4096.0, low=4.0, high=4.0), 1, b"low"),
    (dict(magnitude=math.inf), 1, b"magnitude"), (dict(magnitude=math.nan), 1, b"magnitude"),
    (dict(frequencies=(ctypes.c_double * 32)(*[math.inf] * 32)), 1, b"frequencies"),
])
def test_rope_config_refusals(change, status, message):
    L, out = _lib(), ctypes.c_void_p(1)
    assert L.bbh_rope_create(ctypes.byref(_rope_config(**change)), ctypes.byref(out)) == status
    assert message in L.bbh_last_error() and not out.value
    assert L.bbh_rope_create(None, ctypes.byref(out)) == 1
    assert L.bbh_rope_frequencies(None, None) == 1
    assert L.bbh_rope_free(None) == 0


def _frequencies64(rot, base, scaling="none", factor=1.0, original=0.0, low=0.0, high=0.0):
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "ramp":
        def d(n):
            return rot * math.log(original / (2 * math.pi * n)) / (2 * math.log(base))
        a, b = (min(max(x, 0), rot - 1) for x in (math.floor(d(high)), math.ceil(d(low))))
        r = [min(max((i - a) / max(b - a, 0.001), 0), 1) for i in range(rot // 2)]
        return [x * (1 - y) + x / factor * y for x, y in zip(f, r)]
    if scaling == "bands":
        s = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0), 1) for x in f]
        return [x * y + x / factor * (1 - y) for x, y in zip(f, s)]
    return f


SCALED = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
          dict(scaling="ramp", factor=40.0, original=4096.0, low=1.0, high=32.0),
          dict(scaling="ramp", factor=2.0, original=3.0, low=1.0, high=2.0),  # one step
          dict(scaling="bands", factor=8.0, original=8192.0, low=1.0, high=4.0)]


@pytest.mark.parametrize("kw", SCALED)
@pytest.mark.parametrize("rot", [2, 6, 64, 128, 256])
def test_rope_frequencies(rot, kw):
    from bbh import engine

    rope = engine.Rope(rot, base=10000.0, **kw)
    want = np.array(_frequencies64(rot, 10000.0, **kw))
    np.testing.assert_allclose(rope.frequencies(), want, rtol=1e-13)
    own = engine.Rope(rot, frequencies=want[::-1])
    assert np.array_equal(own.frequencies(), want[::-1])
    own.close()
    own.close()
    with pytest.raises(ValueError):
        engine.Rope(rot, frequencies=want[:-1] if rot > 2 else [1.0, 2.0])
    with pytest.raises(ValueError):
        engine.Rope(rot, scaling="other")


def _rope_args(**change):
    """q, k, v of fused rows of 12 + 4 + 4 heads of 64 at P, outputs apart."""
    from bbh import capi

    a = dict(rows=10, seq=0, heads=12, kv_heads=4, head_dim=64, eps=1e-6, positions=8 * P,
             kv_rows=None, kv_out_rows=0, q_gamma=9 * P, k_gamma=9 * P + 4096)
    for i, (n, h) in enumerate((("q", 0), ("k", 12), ("v", 16))):
        a.update({f"{n}_data": P + h * 128, f"{n}_row": 1280, f"{n}_head": 64})
        a.update({f"{n}_out_data": (2 + i) * P, f"{n}_out_row": (768, 256, 256)[i], f"{n}_out_head": 64})
    a.update(change)
    return capi.RopeArgs(**a)


@pytest.mark.parametrize("change, status, message", [
    (dict(q_data=None), 1, b"null"), (dict(q_out_data=None), 1, b"null"),
    (dict(k_out_data=None), 1, b"together"), (dict(v_data=None), 1, b"together"),
    (dict(rows=-1), 1, b"rows"), (dict(heads=0), 1, b"heads"), (dict(kv_heads=0), 1, b"heads"),
    (dict(head_dim=0), 1, b"head_dim"), (dict(head_dim=257), 7, b"256"),
    (dict(heads=70000), 7, b"65536"), (dict(head_dim=62), 1, b"rot_dim"),
    (dict(positions=None), 1, b"seq"), (dict(eps=-1.0), 1, b"eps"), (dict(eps=math.nan), 1, b"eps"),
    (dict(k_data=None, k_out_data=None), 1, b"k_gamma"),
    (dict(kv_rows=7 * P, kv_out_rows=-1), 1, b"kv_out_rows"),
    (dict(q_row=-8), 1, b"strides"), (dict(k_out_head=-8), 1, b"strides"),
    (dict(q_data=P + 1), 1, b"aligned"), (dict(k_gamma=9 * P + 1), 1, b"aligned"),
    (dict(positions=8 * P + 2), 1, b"aligned"), (dict(kv_rows=7 * P + 4, kv_out_rows=9), 1, b"aligned"),
    (dict(q_out_head=32), 1, b"overlap"), (dict(k_out_row=128), 1, b"overlap"),
    (dict(k_out_data=2 * P), 1, b"outputs overlap"), (dict(v_out_data=2 * P + 1024), 1, b"overlap"),
    # over q, but with other strides, or shifted
    (dict(q_out_data=P, q_out_row=1344), 1, b"overlaps an input"),
    (dict(q_out_data=P + 64, q_out_row=1280), 1, b"overlaps an input"),
    # in place with kv_rows; over the other's columns
    (dict(k_out_data=P + 12 * 128, k_out_row=1280, kv_rows=7 * P, kv_out_rows=10), 1, b"overlaps an input"),
    (dict(k_out_data=P + 16 * 128, k_out_row=1280), 1, b"overlaps an input"),
    (dict(q_out_data=8 * P - 64), 1, b"overlaps an input"),
    (dict(q_out_data=9 * P + 64), 1, b"overlaps an input"),
])
def test_rope_refusals(change, status, message):
    from bbh import engine

    L, rope = _lib(), engine.Rope(64)
    assert L.bbh_rope_heads(rope.handle, ctypes.byref(_rope_args(**change)), None) == status
    assert message in L.bbh_last_error(), L.bbh_last_error()
    assert L.bbh_rope_heads(rope.handle, None, None) == 1


def test_rope_in_place_and_nothing_to_do():
    """In place over fused rows is no overlap; a call without rows is one that does nothing."""
    from bbh import engine

    L, rope = _lib(), engine.Rope(64)
    a = _rope_args(rows=0, q_out_data=P, q_out_row=1280, k_out_data=P + 12 * 128, k_out_row=1280,
                   v_out_data=P + 16 * 128, v_out_row=1280)
    assert L.bbh_rope_heads(rope.handle, ctypes.byref(a), None) == 0


def _args(**change):
    """2 padded sequences of 40 queries and 50 keys, 8 heads on 2, apart in memory."""
    from bbh import capi

    a = dict(batch=2, q_len=40, k_len=50, heads=8, kv_heads=2, head_dim=64, left=-1, right=-1,
             scale=0.125, cap=0.0)
    for i, (n, h, m) in enumerate((("q", 8, 40), ("k", 2, 50), ("v", 2, 50), ("out", 8, 40))):
        a.update({f"{n}_data": (1 + i) * P, f"{n}_batch": m * h * 64, f"{n}_row": h * 64,
                  f"{n}_head": 64})
    a.update(change)
    return capi.AttendArgs(**a)


@pytest.mark.parametrize("change, status, message", [
    (dict(q_data=None), 1, b"null"), (dict(k_data=None), 1, b"null"), (dict(v_data=None), 1, b"null"),
    (dict(out_data=None), 1, b"null"), (dict(batch=-1), 1, b"negative"), (dict(q_len=-1), 1, b"negative"),
    (dict(k_len=-1), 1, b"negative"), (dict(heads=0), 1, b"positive"), (dict(kv_heads=0), 1, b"positive"),
    (dict(head_dim=0), 1, b"positive"), (dict(kv_heads=3), 1, b"multiple"),
    (dict(head_dim=60), 7, b"multiple of 8"), (dict(head_dim=264), 7, b"256"),
    (dict(q_len=1 << 28), 7, b"2^28"), (dict(k_len=(1 << 28) + 1), 7, b"2^28"),
    (dict(batch=1 << 28), 7, b"2^31"), (dict(scale=0.0), 1, b"scale"), (dict(scale=-1.0), 1, b"scale"),
    (dict(scale=math.nan), 1, b"scale"), (dict(scale=math.inf), 1, b"scale"), (dict(cap=-1.0), 1, b"cap"),
    (dict(cap=math.nan), 1, b"cap"), (dict(cap=math.inf), 1, b"cap"),
    (dict(table=6 * P, table_half=-1), 1, b"table_half"),
    (dict(q_offsets=6 * P, q_rows=-1), 1, b"rows"), (dict(k_offsets=6 * P, k_rows=-1), 1, b"rows"),
    (dict(q_data=P + 8), 1, b"16-byte"), (dict(out_data=4 * P + 2), 1, b"16-byte"),
    (dict(k_row=-8), 1, b"negative"), (dict(k_row=132), 1, b"multiples of 8"),
    (dict(v_head=68), 1, b"multiples of 8"), (dict(q_batch=12), 1, b"multiples of 8"),
    (dict(k_row=1 << 23), 7, b"2^23"), (dict(mask=6 * P + 2), 1, b"4-byte"),
    (dict(slopes=6 * P + 1), 1, b"4-byte"), (dict(scratch=6 * P + 8, scratch_bytes=64), 1, b"scratch"),
    (dict(out_head=32), 1, b"overlap"), (dict(out_row=256), 1, b"overlap"),
    (dict(out_batch=64), 1, b"overlap"), (dict(out_data=P), 1, b"overlaps an input"),
    (dict(out_data=2 * P + 1024), 1, b"overlaps an input"),
    (dict(scratch=4 * P, scratch_bytes=1 << 20), 1, b"scratch overlaps"),
])
def test_attend_refusals(change, status, message):
    L = _lib()
    assert L.bbh_attend(ctypes.byref(_args(**change)), None) == status
    assert message in L.bbh_last_error(), L.bbh_last_error()
    assert L.bbh_attend(None, None) == 1


def test_attend_nothing_to_do_and_scratch():
    L = _lib()
    assert L.bbh_attend(ctypes.byref(_args(batch=0)), None) == 0
    assert L.bbh_attend(ctypes.byref(_args(q_len=0)), None) == 0
    assert L.bbh_attend_scratch(None) == 0
    assert L.bbh_attend_scratch(ctypes.byref(_args(head_dim=7))) == 0
    assert L.bbh_attend_scratch(ctypes.byref(_args(batch=0))) == 0
    # a token over a long cache: split; thousands of sequences: not
    assert L.bbh_attend_scratch(ctypes.byref(_args(batch=1, q_len=1, k_len=100000))) > 0
    assert L.bbh_attend_scratch(ctypes.byref(_args(batch=5000, q_len=40, k_len=50))) == 0


def test_python_refuses_host_tensors():
    import torch
    from bbh import engine

    x = torch.zeros(4, 2, 64).half()
    with pytest.raises(TypeError):
        engine.launch_rope(None, x)
    with pytest.raises(TypeError):
        engine.launch_attend(x[None], x[None], x[None], x[None])


# ---- GPU: rotary positions ---------------------------------------------------------

def _gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(torch, g, *shape):
    return torch.randn(shape, device="cuda", generator=g).half()


def _rope64(torch, x, positions, freq, interleaved, magnitude, gamma, eps):
    """The formula in 64 bits, and what a result may be off by."""
    x = x.double()
    if gamma is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    out, size = x.clone(), x.abs()
    f = torch.tensor(freq, device="cuda", dtype=torch.float64)
    rot = 2 * len(freq)
    t = (positions.double()[:, None] * f)[:, None]
    c, s = magnitude * t.cos(), magnitude * t.sin()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    if rot:
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
        both = (x[..., a].abs() + x[..., b].abs()) * abs(magnitude)
        size[..., a], size[..., b] = both, both
    # one rounding to fp16; in fp32 the norm (the sum's tree, rsqrt, two products: < 24 u),
    # sine and cosine (4 u, and a position's own 2^-31 turns), two products and a sum (3 u)
    return out, H * out.abs() + (24 + 4 + 3 + 1) * U * size + TINY


ROPES = [  # rows, heads, kv_heads, dim, rot, interleaved
    (1, 1, 1, 32, 32, False), (3, 5, 2, 64, 64, True), (17, 12, 4, 128, 128, False),
    (33, 7, 7, 80, 48, False), (2, 16, 8, 256, 256, True), (500, 3, 1, 256, 64, False),
    (70, 40, 8, 96, 32, True), (5, 2, 1, 16, 16, False), (6, 3, 3, 8, 0, False), (9, 33, 1, 24, 16, True),
    # no multiples of 8 (heads) or 16 (rotated)
    (13, 5, 3, 40, 20, False), (11, 4, 2, 33, 32, False), (19, 3, 1, 255, 254, True), (4, 2, 2, 2, 2, False),
    (23, 6, 2, 1, 0, False), (5000, 12, 12, 32, 32, False), (21, 8, 2, 100, 70, True),
]


@gpu
@pytest.mark.parametrize("rows,heads,kv,dim,rot,interleaved", ROPES)
@pytest.mark.parametrize("norm", [False, True])
def test_rope(torch_cuda, rows, heads, kv, dim, rot, interleaved, norm):
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, rows + dim + norm)
    qkv = _normal(torch, g, rows, heads + 2 * kv, dim)
    q, k, v = qkv.split((heads, kv, kv), dim=1)
    # far, negative and the outermost positions
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows,), device="cuda", generator=g).int()
    pos[: rows // 2] = torch.arange(rows // 2, device="cuda", dtype=torch.int32)
    pos[-1] = 2 ** 31 - 1
    freq = _frequencies64(rot, 10000.0)
    rope = engine.Rope(rot, interleaved=interleaved, magnitude=1.25) if rot else None
    gammas = [None, None]
    if norm:
        gammas = [(0.5 + torch.rand(dim, device="cuda", generator=g)).half() for _ in range(2)]
    slots = 2 * rows + 1
    nan = float("nan")
    qo = torch.full((rows, heads, dim), nan, device="cuda").half()
    ko = torch.full((slots, kv, dim), nan, device="cuda").half()
    vo = ko.clone()
    to = torch.randperm(slots, device="cuda", generator=g)[:rows].clone()
    lost = rows > 2
    if lost:
        to[0], to[1] = -1, slots  # padding
    seq = 3
    positions = pos if rows != 17 else None
    if positions is None:
        pos = torch.arange(rows, device="cuda", dtype=torch.int32) % seq
    before = qkv.clone()
    engine.launch_rope(rope, q, qo, k=k, k_out=ko, v=v, v_out=vo, positions=positions, seq=seq,
                       q_gamma=gammas[0], k_gamma=gammas[1], eps=1e-5, kv_rows=to)
    torch.cuda.synchronize()
    assert torch.equal(qkv, before)
    magnitude = 1.25 if rot else 1.0
    for got, x, gamma in ((qo, q, gammas[0]), (ko[to.clamp(0, slots - 1)], k, gammas[1])):
        want, tol = _rope64(torch, x, pos, freq, interleaved, magnitude, gamma, 1e-5)
        keep = slice(2, None) if lost and got is not qo else slice(None)
        assert bool(((got.double() - want).abs() <= tol)[keep].all())
    keep = to[2:] if lost else to
    assert torch.equal(vo[keep], v[2:] if lost else v)
    rest = torch.ones(slots, dtype=torch.bool, device="cuda")
    rest[keep] = False
    assert bool(ko[rest].isnan().all()) and bool(vo[rest].isnan().all())
    # in place over the fused rows: the same bits, the values' columns left alone
    engine.launch_rope(rope, q, k=k, positions=positions, seq=seq, q_gamma=gammas[0],
                       k_gamma=gammas[1], eps=1e-5)
    torch.cuda.synchronize()
    assert torch.equal(q, qo) and torch.equal(v, before[:, heads + kv:])
    assert torch.equal(k[2:] if lost else k, ko[keep])


@gpu
@pytest.mark.parametrize("dim,rot", [(64, 32), (48, 16), (40, 22)])
def test_rope_leaves_the_rest_as_it_is(torch_cuda, dim, rot):
    """Values that do not turn pass bit for bit: infinities, NaN and negative zeros too; a
    NaN spoils its own pair only."""
    from bbh import engine

    torch = torch_cuda
    x = torch.randn(3, 2, dim, device="cuda").half()
    x[0, 0, rot] = math.inf
    x[0, 1, dim - 1] = math.nan
    x[1, 0, rot + 1] = -0.0
    x[2, 0, 0] = math.nan
    rope = engine.Rope(rot)
    y = torch.empty_like(x)
    engine.launch_rope(rope, x, y, seq=3)
    torch.cuda.synchronize()
    assert torch.equal(x[..., rot:].view(torch.int16), y[..., rot:].view(torch.int16))
    bad = y.isnan()
    assert bad[2, 0, 0] and bad[2, 0, rot // 2] and int(bad.sum()) == 3


@gpu
def test_rope_other_strides_and_odd_addresses(torch_cuda):
    """Heads before rows, gaps, addresses on 2 bytes: the bits of contiguous operands within
    the tolerance (the two kernels add a norm's squares in another order)."""
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, 5)
    rows, heads, dim = 37, 6, 64
    x = _normal(torch, g, rows, heads, dim)
    gamma = torch.ones(dim, device="cuda").half()
    rope = engine.Rope(dim)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32) * 1000
    want, tol = _rope64(torch, x, pos, _frequencies64(dim, 10000.0), False, 1.0, gamma, 1e-6)

    def put(t, start, *strides):
        room = torch.full((rows * heads * dim * 3 + 64,), float("nan"), device="cuda").half()
        y = room[start:].as_strided((rows, heads, dim), strides)
        if t is not None:
            y.copy_(t)
        return y, room

    for start, strides in ((0, (dim, rows * dim, 1)), (8, (heads * dim + 16, dim, 1)),
                           (1, (heads * dim, dim, 1)), (0, (heads * (dim + 1), dim + 1, 1))):
        xs, _ = put(x, start, *strides)
        ys, room = put(None, start, *strides)
        engine.launch_rope(rope, xs, ys, positions=pos, q_gamma=gamma)
        torch.cuda.synchronize()
        assert bool(((ys.double() - want).abs() <= tol).all()), (start, strides)
        assert int((~room.isnan()).sum()) == x.numel()


@gpu
def test_rope_norm_of_zeros_and_large_values(torch_cuda):
    from bbh import engine

    torch = torch_cuda
    x = torch.zeros(2, 1, 64, device="cuda").half()
    x[1] = 65504.0
    gamma = torch.ones(64, device="cuda").half()
    y = torch.empty_like(x)
    engine.launch_rope(None, x, y, q_gamma=gamma, eps=1e-6)
    torch.cuda.synchronize()
    assert bool((y[0] == 0).all()) and bool((y[1] == 1).all())
    engine.launch_rope(None, x, y, q_gamma=gamma, eps=0.0)
    torch.cuda.synchronize()
    assert bool(y[0].isnan().all()) and bool((y[1] == 1).all())  # 0 / 0


# ---- GPU: attention ---------------------------------------------------------------------

def _attend64(torch, q, k, v, nq, nk, left=-1, right=-1, scale=None, cap=0.0, mask=None, prefix=0,
              slopes=None, table=None):
    """One sequence (its first nq queries, nk keys) in 64 bits, and what a result may be off by."""
    q, k, v = q[:nq].double(), k[:nk].double(), v[:nk].double()
    h, d = q.shape[1:]
    rep = h // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    scale = d ** -0.5 if scale is None else scale
    qt, kt = q.transpose(0, 1), k.permute(1, 2, 0).contiguous()
    s = torch.matmul(qt, kt) * scale
    # fp32 sums of D products
    off = torch.matmul(qt.abs(), kt.abs()) * scale * (d + 4) * U
    if cap:
        s = cap * torch.tanh(s / cap)
        off = off + 16 * cap * U  # exp2, 1 / (1 + e) and the product, of a value up to cap
    dist = torch.arange(nk, device="cuda") - (torch.arange(nq, device="cuda")[:, None] + nk - nq)
    if slopes is not None:
        b = slopes.double()[:, None, None] * dist.abs()
        s, off = s - b, off + 3 * U * b.abs()
    if table is not None:
        half = table.shape[1] // 2
        b = table.double()[:, dist.clamp(-half, half) + half]
        s, off = s + b, off + 3 * U * torch.where(b.isfinite(), b.abs(), 0.0)
    seen = torch.ones_like(dist, dtype=torch.bool)
    if left >= 0:
        seen &= dist >= -left
    if right >= 0:
        seen &= dist <= right
    seen |= torch.arange(nk, device="cuda") < prefix
    if mask is not None:
        seen &= mask[:nk] != 0
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    # seen scores enter as differences from the running maximum, each rounded to fp32
    span = torch.where(s.isfinite(), s.abs(), 0.0)
    off = torch.where(seen, off + 4 * U * span, 0.0).amax(-1, keepdim=True) + \
        4 * U * span.amax(-1, keepdim=True)
    v = v.transpose(0, 1).contiguous()
    out, size = torch.matmul(p, v), torch.matmul(p, v.abs())
    # weights rounded to fp16 (those below 2^-14 of the largest by up to 2^-25 of it), and so
    # their sum; the output rounded once; fp32 sums of nk products in some order
    tol = H * out.abs() + size * (2 * H + 2 * off + 2 * (nk ** 0.5 + 40) * U) + \
        2 * TINY * torch.matmul((p > 0).double() + (s > -1e300), v.abs()) + TINY
    return out.transpose(0, 1), tol.transpose(0, 1)


def _check(torch, got, q, k, v, nq, nk, **kw):
    want, tol = _attend64(torch, q, k, v, nq, nk, **kw)
    d = (got[:nq].double() - want).abs()
    assert bool((d <= tol).all()), (float(d.max()), float((d / tol).max()))


SIZES = [  # batch, q_len, k_len, heads, kv_heads, dim
    (1, 1, 1, 1, 1, 8), (2, 1, 500, 12, 12, 64), (3, 7, 7, 4, 2, 32), (1, 33, 33, 3, 1, 40),
    (2, 64, 64, 8, 8, 64), (1, 129, 129, 5, 1, 96), (2, 100, 300, 6, 2, 128), (1, 257, 257, 4, 4, 72),
    (1, 511, 511, 2, 1, 256), (2, 1, 1000, 8, 1, 256), (1, 31, 2000, 1, 1, 128), (3, 2, 65, 32, 8, 128),
    (1, 5, 4097, 7, 1, 80), (1, 300, 20, 2, 2, 64), (2, 17, 130, 16, 4, 16), (1, 1025, 1025, 2, 1, 128),
    (40, 20, 20, 3, 3, 64), (1, 8, 640, 8, 1, 192),
]
FORMS = [
    dict(), dict(right=0), dict(left=20, right=10), dict(cap=3.0, right=0), dict(slopes=True),
    dict(table=5, left=100), dict(table=40, slopes=True, cap=20.0, right=0), dict(mask=0.6),
    dict(mask=0.1, right=0, prefix=9), dict(prefix=70, right=0, left=12), dict(left=0, right=0),
    dict(mask=0.0), dict(scale=2.0), dict(cap=50.0, mask=0.5, left=30),
]


@gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(f"{k}={v}" for k, v in f.items()) or "plain")
@pytest.mark.parametrize("batch,q_len,k_len,heads,kv,dim", SIZES)
def test_attend(torch_cuda, batch, q_len, k_len, heads, kv, dim, form):
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, q_len + k_len + dim)
    q = _normal(torch, g, batch, q_len, heads, dim)
    k, v = _normal(torch, g, batch, k_len, kv, dim), _normal(torch, g, batch, k_len, kv, dim)
    kw = dict(form)
    if "slopes" in kw:
        kw["slopes"] = torch.rand(heads, device="cuda", generator=g)
    if "table" in kw:
        kw["table"] = torch.randn(heads, 2 * kw["table"] + 1, device="cuda", generator=g)
    mask = prefix = None
    if "mask" in kw:
        share = kw.pop("mask")
        mask = (torch.rand(batch, k_len, device="cuda", generator=g) < share).int() * 7
    if "prefix" in kw:
        prefix = torch.full((batch,), kw.pop("prefix"), device="cuda", dtype=torch.int32)
        prefix[0] = k_len + 3  # past the keys: all of them
    scratch = torch.empty(1 << 22, device="cuda")
    for sc in (None, scratch):
        out = torch.full_like(q, float("nan"))
        engine.launch_attend(q, k, v, out, mask=mask, prefix=prefix, scratch=sc, **kw)
        torch.cuda.synchronize()
        for b in range(batch):
            _check(torch, out[b], q[b], k[b], v[b], q_len, k_len, mask=None if mask is None else mask[b],
                   prefix=0 if prefix is None else min(int(prefix[b]), k_len), **kw)

"""Calls of rotary positions and attention (include/bbh_attend.h) at the edges of what
the header allows: layouts, bit patterns, sizes that no memory holds."""

import ctypes

import pytest

from test_attend import _args, _frequencies64, _gen, _lib, _normal, _rope64, _rope_args, _rope_config

gpu = pytest.mark.gpu


@pytest.mark.parametrize("magnitude", [1e39, -1e300])
def test_a_magnitude_past_fp32_is_refused(magnitude):
    """Finite in double, infinite as the kernels hold it."""
    L, out = _lib(), ctypes.c_void_p(1)
    assert L.bbh_rope_create(ctypes.byref(_rope_config(magnitude=magnitude)), ctypes.byref(out)) == 1
    assert b"magnitude" in L.bbh_last_error() and not out.value
    ok = _rope_config(magnitude=3e38)
    assert L.bbh_rope_create(ctypes.byref(ok), ctypes.byref(out)) == 0 and L.bbh_rope_free(out) == 0


def test_scratch_for_more_rows_than_the_longest_sequences_have():
    """Rows of a packed tensor behind the sequences do not change what it pays to have, however
    many there are."""
    L = _lib()
    kw = dict(batch=1, q_len=300, k_len=100000, heads=8, kv_heads=4, q_offsets=1 << 40)
    want = L.bbh_attend_scratch(ctypes.byref(_args(q_rows=300, **kw)))
    assert want > 0
    for rows in (301, 1 << 31, 1 << 62, (1 << 63) - 1):
        assert L.bbh_attend_scratch(ctypes.byref(_args(q_rows=rows, **kw))) == want, rows


@gpu
def test_queries_without_heads_are_refused(torch_cuda):
    """Not passed over with the keys beside them unturned."""
    from bbh import engine

    torch = torch_cuda
    q = torch.empty(5, 0, 64, device="cuda").half()
    k = torch.randn(5, 2, 64, device="cuda").half()
    with pytest.raises((ValueError, engine.BBHError)):
        engine.launch_rope(engine.Rope(64), q, k=k, k_out=torch.empty_like(k), seq=5)
    assert engine.launch_rope(engine.Rope(64), q, seq=5) is q


@gpu
@pytest.mark.parametrize("dim", [64, 33, 1])
def test_every_bit_pattern_is_moved(torch_cuda, dim):
    """v, and what of q and k neither turns nor is normed: signalling NaN too."""
    from bbh import engine

    torch = torch_cuda
    bits = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16)
    rows = -(-65536 // (2 * dim))
    x = bits.repeat(2)[:rows * 2 * dim].view(rows, 2, dim).view(torch.float16).clone()
    q, k, v = x.clone(), x.clone(), x.clone()
    for gamma in (None, torch.ones(dim, device="cuda").half()):
        outs = [torch.zeros_like(x) for _ in range(3)]
        engine.launch_rope(None, q, outs[0], k=k, k_out=outs[1], v=v, v_out=outs[2], q_gamma=gamma)
        torch.cuda.synchronize()
        for got in outs[1 if gamma is not None else 0:]:
            assert torch.equal(got.view(torch.int16), x.view(torch.int16))
    if dim > 2:
        rot = 2
        y = torch.zeros_like(x)
        engine.launch_rope(engine.Rope(rot), q, y, seq=1)
        torch.cuda.synchronize()
        assert torch.equal(y[..., rot:].view(torch.int16), x[..., rot:].view(torch.int16))


@gpu
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 0, 1)])
@pytest.mark.parametrize("rows,heads,dim", [(7, 3, 64), (50, 12, 64), (5, 2, 40)])
def test_fused_rows_with_a_heads_q_k_and_v_side_by_side(torch_cuda, rows, heads, dim, order):
    """In place: the heads of q, k and v interleave, and overlap nothing."""
    from bbh import engine

    torch = torch_cuda
    g = _gen(torch, rows)
    qkv = _normal(torch, g, rows, heads, 3, dim)
    before = qkv.clone()
    iq, ik, iv = order
    rope = engine.Rope(dim)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    engine.launch_rope(rope, qkv[:, :, iq], k=qkv[:, :, ik], positions=pos)
    torch.cuda.synchronize()
    for i in (iq, ik):
        want, tol = _rope64(torch, before[:, :, i], pos, _frequencies64(dim, 10000.0), False, 1.0, None, 0)
        assert bool(((qkv[:, :, i].double() - want).abs() <= tol).all())
    assert torch.equal(qkv[:, :, iv], before[:, :, iv])
    # q's heads of one key/value head, then its key and value
    group = _normal(torch, g, rows, heads, 4, dim)
    before = group.clone()
    # (heads of a head's group have no one stride: a call for each of them)
    for i in (0, 1):
        engine.launch_rope(rope, group[:, :, i], k=group[:, :, 2] if i == 0 else None, positions=pos)
    torch.cuda.synchronize()
    for i in (0, 1, 2):
        want, tol = _rope64(torch, before[:, :, i], pos, _frequencies64(dim, 10000.0), False, 1.0, None, 0)
        assert bool(((group[:, :, i].double() - want).abs() <= tol).all())
    assert torch.equal(group[:, :, 3], before[:, :, 3])


@pytest.mark.parametrize("change", [
    dict(k_out_data=(1 << 30) + 64, k_out_head=192),       # k's first half over q's second
    dict(k_out_data=(1 << 30) + 2 * 128, k_out_head=128),  # another stride
    dict(k_out_data=(1 << 30) + 128, k_out_head=192, k_out_row=192 * 13),
    dict(k_out_data=(1 << 30) + 12 * 192 * 2 - 64, k_out_head=192, k_out_row=192 * 12),
])
def test_heads_that_do_overlap_are_refused(change):
    from bbh import engine

    p = 1 << 30
    a = dict(q_out_data=p, q_out_head=192, q_out_row=192 * 12, k_out_row=192 * 12, kv_heads=12,
             q_data=20 * p, q_row=768, q_head=64, k_data=21 * p, k_row=768, k_head=64, v_data=None,
             v_out_data=None)
    a.update(change)
    L = _lib()
    assert L.bbh_rope_heads(engine.Rope(64).handle, ctypes.byref(_rope_args(**a)), None) == 1
    assert b"overlap" in L.bbh_last_error()


def _placed(torch, rng, shape, align):
    """An fp16 tensor of this shape with gaps between rows and heads, and its room of NaN."""
    *outer, heads, dim = shape
    head = dim + align * rng.choice((0, 0, 1, 3))
    row = heads * head + align * rng.choice((0, 0, 2, 5))
    if rng.random() < 0.2 and heads > 1:  # heads before rows
        head, row = outer[-1] * (dim + (-dim) % align), dim + (-dim) % align
    size = (outer[-1] - 1) * row + (heads - 1) * head + dim + (-dim) % align
    batch = size + (-size) % align + align * rng.choice((0, 1))
    strides = ([batch] if len(outer) == 2 else []) + [row, head, 1]
    start = align * rng.choice((0, 0, 1, 4))
    room = torch.full((start + batch * (outer[0] if len(outer) == 2 else 1) + align,), float("nan"),
                      device="cuda").half()
    return room[start:].as_strided(shape, strides), room


@gpu
@pytest.mark.parametrize("seed", range(120))
def test_any_call_of_attend(torch_cuda, seed):
    """Lengths, layouts, groups, masks and biases at random, each side padded or packed: every
    sequence as alone, what is behind it left as it was, nothing behind the keys read."""
    import random

    from bbh import engine
    from test_attend import _attend64

    torch, rng = torch_cuda, random.Random(seed)
    g = _gen(torch, seed)
    dim = 8 * rng.randint(1, 32)
    kv = rng.choice((1, 1, 2, 3, 5))
    heads = kv * rng.choice((1, 1, 2, 3, 5, 8, 17, 24, 40))
    batch = rng.choice((1, 2, 3, 7, 40))
    q_most, k_most = rng.choice((1, 1, 2, 5, 33, 70, 300)), rng.choice((1, 9, 64, 65, 130, 513, 1500))
    if batch * heads * q_most * k_most > 3e7:
        batch = 1
    nq = [rng.choice((q_most, rng.randint(0, q_most))) for _ in range(batch)]
    nk = [rng.choice((k_most, rng.randint(0, k_most))) for _ in range(batch)]
    kw, calls = {}, [{} for _ in range(batch)]

    def side(lens, most, n, packed):
        if packed:
            first = rng.choice((0, 3))
            starts = [first]
            for m in lens:
                starts.append(starts[-1] + m)
            t, room = _placed(torch, rng, (starts[-1] + rng.choice((0, 1, 4)) or 1, n, dim), 8)
            return t, room, [slice(a, b) for a, b in zip(starts, starts[1:])], \
                torch.tensor(starts, device="cuda", dtype=torch.int32)
        t, room = _placed(torch, rng, (batch, most, n, dim), 8)
        return t, room, [(b, slice(0, m)) for b, m in enumerate(lens)], None

    qp, kp = rng.random() < 0.5, rng.random() < 0.5
    state = rng.getstate()
    q, _, at_q, q_off = side(nq, q_most, heads, qp)
    rng.setstate(state)  # (the same offsets)
    out, room, _, _ = side(nq, q_most, heads, qp)
    state = rng.getstate()
    k, _, at_k, k_off = side(nk, k_most, kv, kp)
    rng.setstate(state)
    v, _, _, _ = side(nk, k_most, kv, kp)
    for t, at in ((q, at_q), (k, at_k), (v, at_k)):
        for a in at:
            t[a] = torch.randn(t[a].shape, device="cuda", generator=g).half()
    if qp:
        kw.update(q_offsets=q_off, q_len=q_most)
    else:
        kw["q_lengths"] = torch.tensor(nq, device="cuda", dtype=torch.int32)
    if kp:
        kw.update(k_offsets=k_off, k_len=min(k_most, k.shape[0]))
    else:
        kw["k_lengths"] = torch.tensor(nk, device="cuda", dtype=torch.int32)
    k_len = kw.get("k_len", k_most)
    both = {}
    if rng.random() < 0.4:
        both["right"] = rng.choice((0, 0, 3, 100))
    if rng.random() < 0.4:
        both["left"] = rng.choice((0, 7, 64, 200))
    if rng.random() < 0.4:
        both["cap"] = rng.choice((0.5, 5.0, 50.0, 300.0, 1e5))
    if rng.random() < 0.3:
        both["slopes"] = 0.3 * torch.rand(heads, device="cuda", generator=g)
    if rng.random() < 0.3:
        both["table"] = torch.randn(heads, 2 * rng.choice((0, 5, 90, 2500)) + 1, device="cuda", generator=g)
    if rng.random() < 0.3:
        both["scale"] = rng.choice((0.02, 0.3))
    kw.update(both)
    if rng.random() < 0.3:
        mask = (torch.rand(batch, k_len, device="cuda", generator=g) < rng.choice((0.05, 0.6))).int()
        kw["mask"] = mask
        for b in range(batch):
            calls[b]["mask"] = mask[b]
    if rng.random() < 0.3:
        prefix = [rng.choice((0, 5, 64, 100, k_most)) for _ in range(batch)]
        kw["prefix"] = torch.tensor(prefix, device="cuda", dtype=torch.int32)
        for b in range(batch):
            calls[b]["prefix"] = min(prefix[b], nk[b])
    if rng.random() < 0.6:
        kw["scratch"] = torch.empty(rng.choice((100, 100000, 1 << 22)) * 4, device="cuda")
    engine.launch_attend(q, k, v, out, **kw)
    torch.cuda.synchronize()
    written = 0
    for b in range(batch):
        want, tol = _attend64(torch, q[at_q[b]], k[at_k[b]], v[at_k[b]], nq[b], nk[b], **both, **calls[b])
        d = (out[at_q[b]].double() - want).abs()
        assert bool((d <= tol).all()), (b, nq[b], nk[b], dim, heads, kv, sorted(kw), both)
        written += want.numel()
    assert int((~room.isnan()).sum()) == written


@gpu
@pytest.mark.parametrize("seed", range(100))
def test_any_call_of_rope(torch_cuda, seed):
    """Heads, sizes, strides, addresses and slots at random."""
    import random

    from bbh import engine

    torch, rng = torch_cuda, random.Random(seed)
    g = _gen(torch, seed)
    align = rng.choice((1, 2, 4, 8, 8))
    dim = rng.choice((rng.randint(1, 256), 2 * rng.randint(1, 128), 8 * rng.randint(1, 32), 16 * rng.randint(1, 16)))
    rot = min(dim // 2 * 2, rng.choice((0, 2, 16, 64, 256, 2 * rng.randint(0, 128), 16 * rng.randint(0, 16))))
    heads, kv = rng.choice((1, 3, 12, 33, 200)), rng.choice((1, 2, 5, 70))
    rows = rng.choice((1, 2, 19, 130, 1000, 3000))
    if rows * (heads + 2 * kv) * dim > 1 << 24:
        rows = 5
    interleaved, norms = rng.random() < 0.5, (rng.random() < 0.5, rng.random() < 0.5)
    slots = rows + rng.choice((0, 7)) if rng.random() < 0.4 else None
    xs, ys, rooms = [], [], []
    for n, n_out in ((heads, rows), (kv, slots or rows), (kv, slots or rows)):
        x, _ = _placed(torch, rng, (rows, n, dim), align)
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        y, room = _placed(torch, rng, (n_out, n, dim), align)
        xs.append(x), ys.append(y), rooms.append(room)
    freq = _frequencies64(rot, 10000.0)
    rope = engine.Rope(rot, interleaved=interleaved) if rot else None
    gammas = [(0.5 + torch.rand(dim, device="cuda", generator=g)).half() if n else None for n in norms]
    pos = torch.randint(-100000, 1000000, (rows,), device="cuda", generator=g).int()
    seq, positions = rng.randint(1, 50), pos if rng.random() < 0.7 else None
    if positions is None:
        pos = torch.arange(rows, device="cuda", dtype=torch.int32) % seq
    to = torch.randperm(slots, device="cuda", generator=g)[:rows].clone() if slots else None
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    if slots and rows > 2:
        to[0], to[1] = -5, slots
        keep[:2] = False
    engine.launch_rope(rope, xs[0], ys[0], k=xs[1], k_out=ys[1], v=xs[2], v_out=ys[2], positions=positions,
                       seq=seq, q_gamma=gammas[0], k_gamma=gammas[1], eps=1e-5, kv_rows=to)
    torch.cuda.synchronize()
    n = int(keep.sum())
    for i, (x, y) in enumerate(zip(xs[:2], ys)):
        want, tol = _rope64(torch, x, pos, freq, interleaved, 1.0, gammas[i], 1e-5)
        got = y if i == 0 or to is None else y[to.clamp(0, slots - 1)]
        ok = (got.double() - want).abs() <= tol
        assert bool((ok if i == 0 else ok[keep]).all()), (rows, heads, kv, dim, rot, align, norms)
    got = ys[2] if to is None else ys[2][to.clamp(0, slots - 1)]
    assert torch.equal(got[keep], xs[2][keep])
    for room, count in zip(rooms, (rows * heads, n * kv, n * kv)):
        assert int((~room.isnan()).sum()) == count * dim

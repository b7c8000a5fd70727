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

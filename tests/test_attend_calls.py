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

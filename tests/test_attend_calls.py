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

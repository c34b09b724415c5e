"""A table of rotations is not made of frequencies that are no numbers (refused before any device is asked for)."""
import ctypes
import math

import pytest

from jitnn_b200 import _lib
from jitnn_b200.build import build


@pytest.mark.parametrize("at", [0, 15, 31])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_refused(at, bad):
    build()
    L = _lib.load()
    freqs, out = (ctypes.c_double * 32)(*[0.5] * 32), ctypes.c_void_p()
    freqs[at] = bad
    assert L.jq_rope_create(0, 16, 64, freqs, 1.0, 0, ctypes.byref(out)) == _lib.JQ_ERR_INVALID
    assert "frequency %d" % at in _lib.last_error() and not out.value

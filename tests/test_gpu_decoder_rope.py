"""Frequencies of the decoder's rotation that are no numbers are refused, and leave both kinds of caches rotated as they were."""
import ctypes
import math

import numpy as np
import pytest

from jitnn_b200 import _lib
from test_gpu_decoder_pages import build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("paged", [False, True])
def test_frequencies_that_are_no_numbers(paged):
    cfg, _, dec = build(256, 4, 2)
    L, half = _lib.load(), cfg.head_dim // 2
    if paged:
        dec.set_pages(4, 16, "F32")
    tokens = np.arange(12, dtype=np.int32)
    step = (lambda: dec.forward_pages([tokens], [[2]], [12])[0]) if paged else (lambda: dec.forward(tokens, 0)[0])
    want = step()
    freqs = [cfg.rope_base ** (-2.0 * i / cfg.head_dim) for i in range(half)]
    for bad in (math.nan, math.inf, -math.inf):
        for i in (0, half - 1):
            given = freqs[:i] + [bad] + freqs[i + 1:]
            assert L.jq_decoder_set_rope(dec._h, (ctypes.c_double * half)(*given), 1.0) == _lib.JQ_ERR_INVALID
            assert "frequency %d" % i in _lib.last_error()
    assert L.jq_decoder_set_rope(dec._h, (ctypes.c_double * half)(*freqs), math.nan) == _lib.JQ_ERR_INVALID
    assert np.array_equal(step(), want)
    _lib.check(L.jq_decoder_set_rope(dec._h, (ctypes.c_double * half)(*[f / 2 for f in freqs]), 1.0))
    assert not np.array_equal(step(), want)
    _lib.check(L.jq_decoder_set_rope(dec._h, (ctypes.c_double * half)(*freqs), 1.0))
    assert np.array_equal(step(), want)
    dec.close()

"""A call that the device has no memory for fails, and the calls behind it do not fail with it."""
import numpy as np
import pytest
import torch

from jitnn_b200 import Rope
from test_gpu_decoder_pages import build

pytestmark = pytest.mark.gpu


def test_fewer_pages_after_too_many():
    """Pages of terabytes are asked for and not given (nothing is allocated); then as many as there is room for."""
    cfg, _, dec = build(256, 4, 2)
    dec.set_pages(4, 16, "F32")
    tokens = np.arange(9, dtype=np.int32)
    want = dec.forward_pages([tokens], [[2]], [9])[0]
    x = torch.randn(3, 2, 64, device="cuda")
    rope = Rope(50, 64)
    turned = rope.rotate(x, 5)
    for after in (lambda: None, lambda: rope.rotate(x, 5), lambda: Rope(50, 64)):
        with pytest.raises(MemoryError):
            dec.set_pages(2 ** 30, 1024, "F32")
        after()
        dec.set_pages(4, 16, "F32")
        assert np.array_equal(dec.forward_pages([tokens], [[2]], [9])[0], want)
        assert torch.equal(rope.rotate(x, 5), turned)
    dec.close()

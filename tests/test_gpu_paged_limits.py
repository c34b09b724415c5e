"""Paged attention where its waits run out: it returns, leaves a status, and the next call is as good as any."""
import pytest
import torch

from jitnn_b200 import _lib, device_status
from test_gpu_paged import BF16, F16, F32, Setup, normal

pytestmark = pytest.mark.gpu


@pytest.fixture()
def short_waits():
    """A microsecond, which the first keys' copy from memory and the products behind it do not keep."""
    L = _lib.load()
    torch.cuda.synchronize()
    assert device_status(0) == 0
    _lib.check(L.jq_set_option(b"wait_limit_us", 1))
    yield lambda: _lib.check(L.jq_set_option(b"wait_limit_us", 2000000))
    _lib.check(L.jq_set_option(b"wait_limit_us", 2000000))


@pytest.mark.parametrize("act,cache", [(F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,lengths,prefix", [([150, 90], [700, 400], 0), ([100, 3], [100, 60], 900), ([4] * 8, [300] * 8, 9000)])
def test_waits_that_run_out(short_waits, act, cache, hd, rows, lengths, prefix):
    """Own keys by the tile kernel, the prefix with them, and the prefix alone beside the stream kernel. Some pages are missing, so that the tiles' flags are in use."""
    t = Setup(rows, lengths, 2, hd, 16, cache, prefix=prefix, hole=0.0, seed=31)
    q = normal(t.tokens, 32, hd, dtype=act, seed=31).cuda()
    page, last = int(t.tables[0, 2]), t.starts[1] - 1
    for missing in (True, False):
        t.batch.tables[0, 2] = -1 if missing else page
        for _ in range(5):
            t.cache.attention(q, t.batch)
        torch.cuda.synchronize()
        code = device_status(0)  # (of several codes any one is there)
        assert 10 <= code <= 19 or (missing and code == 96)
    short_waits()
    whole = t.cache.attention(q, t.batch)
    torch.cuda.synchronize()
    assert torch.isfinite(whole).all() and device_status(0) == 0
    t.batch.tables[0, 2] = -1
    part = t.cache.attention(q, t.batch)
    torch.cuda.synchronize()
    assert torch.isfinite(part).all() and device_status(0) == 96
    assert torch.equal(whole[last + 1:], part[last + 1:]) and not torch.equal(whole[last], part[last])

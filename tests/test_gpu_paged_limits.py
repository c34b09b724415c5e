"""Paged attention at its limits. Waits that run out: it returns, leaves a status, and the next call is as good as any. Lengths beyond the tables, tables of too many keys."""
import math

import pytest
import torch

import paged_oracle as oracle
from jitnn_b200 import PagedBatch, PagedCache, _lib, device_status
from test_gpu_paged import BF16, F16, F32, Setup, normal, within

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


@pytest.mark.parametrize("act,cache", [(F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("limit", [2, 3, 4, 6, 9, 14])
def test_waits_that_run_out_anywhere(short_waits, act, cache, hd, limit):
    """Limits that the first waits keep and later ones do not, with missing pages and values that are not finite under the rows' masks: whatever gave up, the call behind it is right."""
    t = Setup([130, 150, 5], [900, 1500, 60], 2, hd, 16, cache, prefix=700, hole=float("nan"), seed=33)
    q = normal(t.tokens, 32, hd, dtype=act, seed=33).cuda()
    t.cache.v[int(t.tables[1, 90]), :, 3] = float("inf")  # (a key that some of the second sequence's rows see)
    table = t.batch.tables.clone()
    table[0, 5] = table[1, 70] = -1
    missing = PagedBatch(table, t.batch.starts, t.batch.lengths, prefix=t.batch.prefix, prefix_length=700)
    _lib.check(_lib.load().jq_set_option(b"wait_limit_us", limit))
    for _ in range(10):
        t.cache.attention(q, t.batch)
        t.cache.attention(q, missing)
    torch.cuda.synchronize()
    code = device_status(0)
    assert code == 96 or 10 <= code <= 19
    short_waits()
    for batch, after in ((t.batch, 0), (missing, 96)):
        first = t.cache.attention(q, batch)
        bits = torch.int32 if act is F32 else torch.int16
        assert torch.equal(t.cache.attention(q, batch).view(bits), first.view(bits))
        assert torch.isfinite(first[: t.starts[1]]).all() and not torch.isfinite(first[t.starts[2] - 1]).any()
        torch.cuda.synchronize()
        assert device_status(0) == after


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("hd,rows", [(40, [2, 1]), (96, [1, 1]), (64, [2, 1]), (256, [1, 2]), (128, [40, 1])])
@pytest.mark.parametrize("prefix", [0, 20])
@pytest.mark.parametrize("length", [49, 2 ** 30, 2 ** 31 - 50, 2 ** 31 - 1])
def test_lengths_that_the_table_does_not_have(act, cache, hd, rows, prefix, length):
    """The first sequence names more keys than its three pages hold: it sees all of those, behind the prefix, and leaves a status."""
    t = Setup(rows, [48, 20 if rows[1] < 20 else 40], 2, hd, 16, cache, prefix=prefix, hole=0.0, extra_width=0, seed=32)
    q = normal(t.tokens, 4, hd, dtype=act, seed=32)
    t.batch.lengths[0] = length
    got = t.cache.attention(q.cuda(), t.batch)
    torch.cuda.synchronize()
    assert device_status(0) == 96
    pk, pv = (oracle.keys_of(x, t.prefix, 16, prefix) if prefix else x[:0, :, 0] for x in (t.k, t.v))
    for row, s, at in t.each_row():
        count = at + 1 if s else max(0, min(48, length - (rows[0] - 1 - row)))
        k, v = (torch.cat((p, oracle.keys_of(x, t.tables[s], 16, count))) for p, x in ((pk, t.k), (pv, t.v)))
        want, size, score = oracle.attention(q[row], k, v, 1 / math.sqrt(hd))
        within(got[row], want, oracle.attention_bound(want, size, score, hd, len(k), act, cache), "row %d" % row)


def test_tables_of_more_keys_than_numbers_are_refused():
    k, v = (torch.zeros(1, 1, 1024, 40, device="cuda") for _ in range(2))
    cache = PagedCache(1, 1024, 1, 40, k=k, v=v)
    tables = torch.zeros(1, 2 ** 21, dtype=torch.int32, device="cuda")
    whole = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.zeros(1, 1, 40, device="cuda")
    for width, prefix in ((2 ** 21, 0), (2 ** 21 - 1, 800)):
        batch = PagedBatch(tables[:, :width], whole(0, 1), whole(5), prefix=tables[0, :1], prefix_length=prefix)
        for call in (lambda: cache.attention(x, batch), lambda: cache.append(x, x, x, batch)):
            with pytest.raises(ValueError, match="positions are below"):
                call()
    batch = PagedBatch(tables[:, : 2 ** 21 - 1], whole(0, 1), whole(5), prefix=tables[0, :1], prefix_length=768)
    assert torch.equal(cache.attention(x, batch), x) and torch.equal(cache.append(x, x, x, batch), x)
    assert device_status(0) == 0

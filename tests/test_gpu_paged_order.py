"""Paged attention by two kernels, one for the prefix and one for own keys, behind kernels that write everything it reads: pages, tables, starts, lengths and queries."""
import pytest
import torch

from test_gpu_paged import BF16, F16, F32, Setup, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,cache", [(BF16, BF16), (F16, F16), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("hd,rows,lengths,prefix", [(64, [4] * 8, [60 + 30 * i for i in range(8)], 8200), (128, [1] * 24, [3 + 90 * i for i in range(24)], 4100), (64, [2] * 3, [2, 9, 40], 16000)])
@pytest.mark.parametrize("captured", [False, True])
def test_everything_is_written_just_in_front(act, cache, hd, rows, lengths, prefix, captured):
    t = Setup(rows, lengths, 2, hd, 16, cache, prefix=prefix, hole=0.0, seed=51)
    q = normal(t.tokens, 32, hd, dtype=act, seed=51).cuda()
    want = t.cache.attention(q, t.batch)
    read = [t.cache.k, t.cache.v, t.batch.tables, t.batch.starts, t.batch.lengths, t.batch.prefix, q]
    true = [x.clone() for x in read]
    torch.cuda.synchronize()

    def run():
        got = []
        for turn in range(3):
            for x, y in zip(read, true):
                x.zero_()  # (every id and number is one that the cache has)
            got.append(t.cache.attention(q, t.batch))  # reads all of that, no rows: first-level caches hold it
            for x, y in zip(read if turn else read[::-1], true if turn else true[::-1]):
                x.copy_(y)
            got.append(t.cache.attention(q, t.batch))
        return got

    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run()
        for _ in range(10):
            g.replay()
    else:
        for _ in range(10):
            got = run()
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want if i % 2 else torch.zeros_like(want)), i

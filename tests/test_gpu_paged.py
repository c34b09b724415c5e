"""Rotary positions, append and attention of the paged cache against 64-bit forms, at the sizes, layouts and masks where they can go wrong."""
import math

import pytest
import torch

import paged_oracle as oracle
from jitnn_b200 import PagedBatch, PagedCache, Rope, RopeScaling, device_status

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SCALINGS = {None: None, "linear": RopeScaling.linear(4), "llama3": RopeScaling.llama3(8, 1, 4, 512), "yarn": RopeScaling.yarn(4, 512, 32, 1)}
ORACLE_SCALINGS = {None: None, "linear": ("linear", 4.0), "llama3": ("llama3", 8.0, 1.0, 4.0, 512.0), "yarn": ("yarn", 4.0, 512.0, 32.0, 1.0)}


def normal(*shape, dtype=F32, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype)


def within(got, want, bound, what=""):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all(), what
    worst = int((off - bound).argmax())
    assert (off <= bound).all(), "%s: %g off at %d, at most %g" % (what, off.flatten()[worst], worst, bound.flatten()[worst])


def no_status():
    assert device_status(0) == 0


# ---- rotary positions ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,dim,scaling", [(128, 128, None), (128, 64, "llama3"), (64, 64, "yarn"), (256, 128, "linear"), (80, 80, None), (96, 36, "llama3"), (6, 2, None), (512, 512, "yarn")])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotation(dtype, interleaved, hd, dim, scaling, inverse):
    rope = Rope(4000, dim, base=10000.0, scaling=SCALINGS[scaling], interleaved=interleaved)
    freqs, magnitude = oracle.frequencies(dim, 10000.0, ORACLE_SCALINGS[scaling])
    q, k = normal(5, 3, hd, dtype=dtype, seed=1), normal(5, 2, hd, dtype=dtype, seed=2)
    at = [0, 3999, 17, 511, 17]
    turn = rope.backward if inverse else rope.rotate
    got = turn((q.cuda(), k.cuda()), torch.tensor(at, device="cuda"))
    for x, y in zip((q, k), got):
        for t, position in enumerate(at):
            want, size = oracle.rotated(x[t], position, freqs, magnitude, interleaved, inverse)
            within(y[t], want, oracle.rotation_bound(want, size, dtype))
            assert torch.equal(y[t, :, dim:].cpu(), x[t, :, dim:])  # what is not rotated is copied
    no_status()


@pytest.mark.parametrize("kind", ["int32", "int64", "offset", "rows"])
def test_rotation_positions_of_a_batch(kind):
    rope = Rope(100, 64)
    freqs, magnitude = oracle.frequencies(64)
    x = normal(3, 7, 2, 64)
    if kind == "rows":
        at = torch.randint(0, 100, (3, 7), generator=torch.Generator().manual_seed(4))
        got = rope.rotate(x.cuda(), at.t().contiguous().t().cuda())  # strided
    else:
        at = (torch.arange(7) + 93).expand(3, 7)
        got = rope.rotate(x.cuda(), 93 if kind == "offset" else at[0].to(getattr(torch, kind)).cuda())
    for b in range(3):
        for t in range(7):
            want, size = oracle.rotated(x[b, t], int(at[b, t]), freqs, magnitude, False)
            within(got[b, t], want, oracle.rotation_bound(want, size, F32))


@pytest.mark.parametrize("dtype,hd", [(F32, 128), (BF16, 64), (F16, 72)])
@pytest.mark.parametrize("cut", [0, 1])
def test_rotation_of_slices_in_place(dtype, hd, cut):
    """Queries and keys inside one fused projection, rotated where they are; with a cut of one element, at odd addresses. What is around them stays."""
    rope = Rope(64, hd)
    base = normal(9, 8 * hd + 3, dtype=dtype, seed=5)
    fused = base.cuda()
    q, k = fused[:, cut: cut + 4 * hd].unflatten(1, (4, hd)), fused[:, cut + 4 * hd: cut + 6 * hd].unflatten(1, (2, hd))
    alone = rope.rotate((q.clone(), k.clone()), 20)
    got = rope.rotate((q, k), 20, out=(q, k))
    assert got[0] is q and torch.equal(q, alone[0]) and torch.equal(k, alone[1])
    assert torch.equal(fused[:, :cut].cpu(), base[:, :cut]) and torch.equal(fused[:, cut + 6 * hd:].cpu(), base[:, cut + 6 * hd:])
    transposed = normal(4, 9, hd, dtype=dtype, seed=6).cuda().transpose(0, 1)  # heads outermost
    assert torch.equal(rope.rotate(transposed, 3), rope.rotate(transposed.contiguous(), 3))


def test_rotation_gradient_against_differences():
    rope = Rope(1000, 32, scaling=RopeScaling.yarn(2, 64), interleaved=True)
    freqs, magnitude = oracle.frequencies(32, 10000.0, ("yarn", 2.0, 64.0, 32.0, 1.0))
    x, g = normal(1, 1, 48, seed=7).double(), normal(1, 1, 48, seed=8)
    got = rope.backward(g.cuda(), 77)[0, 0].cpu().double()
    step = 2.0 ** -10  # the rotation is linear: differences of the 64-bit form are exact to its rounding
    for i in range(48):
        up, down = x.clone(), x.clone()
        up[0, 0, i] += step
        down[0, 0, i] -= step
        slope = ((oracle.rotated(up[0], 77, freqs, magnitude, True)[0] - oracle.rotated(down[0], 77, freqs, magnitude, True)[0]) * g[0].double()).sum() / (2 * step)
        assert abs(float(slope - got[i])) <= 8 * 2.0 ** -24 * 2 * float(g.abs().max()) * magnitude + 1e-11


def test_positions_outside_the_table_are_nan_and_leave_a_status():
    rope = Rope(10, 8)
    x = normal(4, 1, 8).cuda()
    got = rope.rotate(x, torch.tensor([9, 10, -1, 2 ** 31 - 1], device="cuda"))
    assert device_status(0) == 97
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1:]).all()
    got = rope.rotate(x, torch.tensor([0, 2 ** 40, -2 ** 40, 9], device="cuda"))
    assert device_status(0) == 97
    assert torch.isfinite(got[[0, 3]]).all() and torch.isnan(got[1:3]).all()
    with pytest.raises(ValueError, match="positions 7 to 10"):
        rope.rotate(x, 7)
    assert rope.rotate(x[:0], 3).shape == (0, 1, 8)


# ---- the cache -----------------------------------------------------------------------------------------------------------------------

class Setup:
    """A batch on a cache: rows and lengths of each sequence, pages in random order, everything that nobody may read set to `hole`."""

    def __init__(self, rows, lengths, kv, hd, page, cache, prefix=0, pad=0, hole=math.nan, seed=0, spare=2, extra_width=1):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lengths, self.page, self.prefix_length = rows, lengths, page, prefix
        n, width, ahead = len(rows), max(1, -(-max(max(lengths), 1) // page)) + extra_width, -(-prefix // page)
        self.pages = n * width + ahead + spare
        order = torch.randperm(self.pages, generator=g).int()
        self.tables, self.prefix = order[: n * width].view(n, width), order[n * width: n * width + ahead]
        self.starts = [sum(rows[:i]) for i in range(n + 1)]
        self.tokens = sum(rows) + pad
        shape = (self.pages, kv, page, hd)
        self.k, self.v = (torch.randn(shape, generator=g).to(cache) for _ in range(2))
        seen = torch.zeros(self.pages, page, dtype=torch.bool)
        for table, count in [(self.tables[s], lengths[s]) for s in range(n)] + [(self.prefix, prefix)]:
            i = torch.arange(count)
            seen[table[i // page].long(), i % page] = True
        for x in (self.k, self.v):
            x.permute(0, 2, 1, 3)[~seen] = hole
        self.seen = seen
        self.cache = PagedCache(self.pages, page, kv, hd, dtype=cache, k=self.k.cuda(), v=self.v.cuda())
        self.batch = PagedBatch(self.tables.cuda(), torch.tensor(self.starts, dtype=torch.int32, device="cuda"), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                prefix=self.prefix.cuda() if ahead else None, prefix_length=prefix)

    def each_row(self):
        """(row, sequence, own position)"""
        for s, n in enumerate(self.rows):
            for i in range(n):
                yield self.starts[s] + i, s, self.lengths[s] - n + i


TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv,hd,dim,interleaved,cut", [(8, 2, 128, 128, False, 0), (4, 4, 64, 32, True, 0), (3, 1, 256, 256, False, 0), (2, 1, 80, 80, True, 0), (6, 3, 34, 18, False, 0), (8, 2, 64, 64, False, 1)])
def test_append(act, cache, heads, kv, hd, dim, interleaved, cut):
    t = Setup([1, 0, 5, 2, 1, 3], [1, 40, 37, 16, 0, 17], kv, hd, 16, cache, prefix=21, pad=3)
    rope = Rope(100, dim, interleaved=interleaved)
    freqs, magnitude = oracle.frequencies(dim)
    base = normal(t.tokens, (heads + 2 * kv) * hd + cut, dtype=act, seed=9)
    fused = base.cuda()[:, cut:].unflatten(1, (heads + 2 * kv, hd))
    q, k, v = fused[:, :heads], fused[:, heads: heads + kv], fused[:, heads + kv:]
    got = t.cache.append(q, k, v, t.batch, rope=rope)
    plain = base[:, cut:].unflatten(1, (heads + 2 * kv, hd))
    stored = torch.zeros_like(t.seen)
    for row, s, at in t.each_row():
        if at < 0:
            assert torch.equal(got[row].cpu(), torch.zeros(heads, hd, dtype=act))
            continue
        want, size = oracle.rotated(plain[row], at + 21, freqs, magnitude, interleaved)
        within(got[row], want[:heads], oracle.rotation_bound(want, size, act)[:heads])
        page, slot = int(t.tables[s, at // 16]), at % 16
        # rounded to the rows' type, then to the pages' where that is another
        bound = oracle.rotation_bound(want, size, act) + (0 if act is cache else oracle.HALF_STEP[cache] * (want.abs() + oracle.rotation_bound(want, size, act)) + oracle.SMALLEST[cache])
        within(t.cache.k[page, :, slot], want[heads: heads + kv], bound[heads: heads + kv])
        assert torch.equal(t.cache.v[page, :, slot].cpu(), plain[row, heads + kv:].to(cache))
        stored[page, slot] = True
    assert torch.equal(got[t.starts[-1]:].cpu(), torch.zeros(3, heads, hd, dtype=act))  # rows of no sequence
    for x, before in ((t.cache.k, t.k), (t.cache.v, t.v)):  # nothing else has changed
        assert torch.equal(x.permute(0, 2, 1, 3).cpu()[~stored].view(torch.uint8), before.permute(0, 2, 1, 3)[~stored].view(torch.uint8))
    kept = normal(t.tokens, heads, hd, dtype=act, seed=10).cuda()
    before = kept.clone()
    assert t.cache.append(q, k, v, t.batch, rope=rope, out=kept) is kept
    assert torch.equal(kept[t.starts[-1]:], before[t.starts[-1]:]) and torch.equal(kept[: t.starts[-1]][:1], got[:1])
    no_status()


def test_append_without_queries_or_rotation():
    t = Setup([2, 1], [20, 3], 2, 64, 16, F32)
    k, v = normal(3, 2, 64, seed=1), normal(3, 2, 64, seed=2)
    assert t.cache.append(None, k.cuda(), v.cuda(), t.batch) is None
    q = normal(3, 4, 64, seed=3)
    assert torch.equal(t.cache.append(q.cuda(), k.cuda(), v.cuda(), t.batch).cpu(), q)
    for row, s, at in t.each_row():
        assert torch.equal(t.cache.k[int(t.tables[s, at // 16]), :, at % 16].cpu(), k[row])


# rows of each sequence, lengths, prefix, page: single tokens; one key; sequences without rows or keys; more rows than keys; ends in front of, at and behind a page's
BATCHES = [([1], [1], 0, 16), ([1], [577], 0, 16), ([1, 1, 1, 1], [15, 16, 17, 0], 0, 16), ([1, 1, 1], [1, 300, 64], 33, 32), ([2, 0, 5, 1], [2, 9, 3, 130], 16, 16),
           ([0, 1, 0], [5, 6, 0], 1, 64), ([17, 3], [40, 65], 64, 64), ([1] * 20, [7 * i for i in range(20)], 129, 16), ([40], [40], 5, 16), ([1, 2], [700, 1100], 2000, 128),
           ([8, 8], [0, 0], 0, 16), ([4, 1], [0, 2], 3, 16), ([33, 70, 1], [600, 71, 9], 300, 16)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (2, 2, 64), (5, 1, 256), (16, 1, 64), (3, 3, 128), (20, 1, 128), (6, 2, 40)])
@pytest.mark.parametrize("at", range(len(BATCHES)))
def test_attention(act, cache, heads, kv, hd, at):
    rows, lengths, prefix, page = BATCHES[at]
    t = Setup(rows, lengths, kv, hd, page, cache, prefix=prefix, pad=at % 3, seed=at)
    q = normal(t.tokens, heads, hd, dtype=act, seed=at) * (3.0 if at % 2 else 1.0)
    check_attention(t, q.to(act), heads, kv, hd, act, cache)


def check_attention(t, q, heads, kv, hd, act, cache, scale=None):
    got = t.cache.attention(q.cuda(), t.batch, scale=scale)
    scale = 1 / math.sqrt(hd) if scale is None else scale
    pk, pv = (oracle.keys_of(x, t.prefix, t.page, t.prefix_length) if t.prefix_length else x[:0, :, 0] for x in (t.k, t.v))
    for row, s, at in t.each_row():
        k, v = (torch.cat((p, oracle.keys_of(x, t.tables[s], t.page, max(0, at + 1)))) for p, x in ((pk, t.k), (pv, t.v)))
        if not len(k):
            assert torch.equal(got[row].cpu(), torch.zeros(heads, hd, dtype=act))
            continue
        want, size, score = oracle.attention(q[row], k, v, scale)
        within(got[row], want, oracle.attention_bound(want, size, score, hd, len(k), act, cache), "row %d" % row)
    assert torch.equal(got[t.starts[-1]:].cpu(), torch.zeros(t.tokens - t.starts[-1], heads, hd, dtype=act))
    no_status()
    return got


@pytest.mark.parametrize("act,cache", TYPES[1:])
@pytest.mark.parametrize("hd,rows,prefix,page", [(64, 4, 3905, 16), (128, 1, 4001, 64), (64, 1, 15700, 128), (64, 4, 8200, 16), (128, 1, 6500, 64)])
def test_attention_behind_a_long_prefix(act, cache, hd, rows, prefix, page):
    """Many products with the prefix's keys, few rows a sequence: on both sides of where the prefix gets a kernel of its own."""
    n = 8 if rows > 1 else 16
    t = Setup([rows] * n, [rows + 11 * i for i in range(n)], 2, hd, page, cache, prefix=prefix, pad=1, seed=21)
    check_attention(t, normal(t.tokens, 32, hd, dtype=act, seed=21), 32, 2, hd, act, cache)


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("rows,lengths,prefix,page", [([500, 1, 40], [500, 1030, 700], 1300, 256), ([3, 2], [1024, 2049], 1025, 1024), ([700], [900], 0, 512)])
def test_attention_of_prompts_and_of_large_pages(act, cache, heads, kv, hd, rows, lengths, prefix, page):
    t = Setup(rows, lengths, kv, hd, page, cache, prefix=prefix, seed=23)
    check_attention(t, normal(t.tokens, heads, hd, dtype=act, seed=23), heads, kv, hd, act, cache)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows,n", [(64, 1, 70), (128, 1, 70), (256, 1, 50), (64, 5, 23), (128, 3, 30)])
def test_attention_of_many_short_sequences(act, cache, hd, rows, n):
    """More runs of keys than workers: where one begins or ends, an item's first runs, its last ones or none of them may be a worker's."""
    t = Setup([rows] * n, [(37 * i) % 290 for i in range(n)], 8, hd, 16, cache, prefix=40 if n == 23 else 0, seed=22)
    heads = 128 if rows > 1 else 8
    check_attention(t, normal(t.tokens, heads, hd, dtype=act, seed=22), heads, 8, hd, act, cache)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_does_not_reach_it(act, cache, hd, bad):
    """The newest keys and values of a run of drafts are not finite: the rows in front of them are what they were, the last sees them.

    Where values are not finite the kernels may add them up one by one, in another order than otherwise: two results that are each within attention_bound of the same 64-bit
    value are within twice that of each other, which is what is asked of the rows (the bits need not be the same)."""
    t = Setup([1, 4, 1], [50, 61, 16], 2, hd, 16, cache, prefix=20, hole=bad, seed=3)
    q = normal(t.tokens, 4, hd, dtype=act, seed=3)
    clean = check_attention(t, q, 4, 2, hd, act, cache)
    rest, bounds = [0, 1, 2, 3, 5], []
    for row, s, at in t.each_row():
        k, v = (torch.cat((oracle.keys_of(x, t.prefix, 16, 20), oracle.keys_of(x, t.tables[s], 16, at + 1))) for x in (t.k, t.v))
        want, size, score = oracle.attention(q[row], k, v, 1 / math.sqrt(hd))
        bounds.append(2 * oracle.attention_bound(want, size, score, hd, len(k), act, cache))
    bounds = torch.stack(bounds)[rest]
    page, slot = int(t.tables[1, 60 // 16]), 60 % 16
    t.cache.k[page, :, slot] = bad
    t.cache.v[page, :, slot] = bad
    got = t.cache.attention(q.cuda(), t.batch)
    within(got[rest], clean[rest].double().cpu(), bounds)
    assert not torch.isfinite(got[4]).any() if not (bad == -math.inf) else True
    t.cache.k[page, :, slot] = 0.0  # only the value is not finite: what sees it is that
    got = t.cache.attention(q.cuda(), t.batch)
    within(got[rest], clean[rest].double().cpu(), bounds)
    assert not torch.isfinite(got[4]).any()
    no_status()


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, F16), (BF16, BF16)])
def test_scores_far_apart(act, cache):
    """Keys of very different size, negative infinite scores among them (a key of -inf against positive queries): such keys weigh nothing; and a scale of one's own."""
    t = Setup([1, 2], [200, 90], 2, 128, 16, cache, prefix=40, seed=5)
    t.cache.k.mul_(30.0)
    t.k = t.cache.k.cpu()
    q = normal(3, 4, 128, dtype=act, seed=5)
    check_attention(t, q, 4, 2, 128, act, cache)
    check_attention(t, q, 4, 2, 128, act, cache, scale=-0.003)
    check_attention(t, q, 4, 2, 128, act, cache, scale=0.0)
    q = q.abs() + 0.5
    for table, i in ((t.tables[0], 3), (t.tables[0], 199), (t.prefix, 7)):
        t.cache.k[int(table[i // 16]), :, i % 16] = -math.inf
        t.cache.v[int(table[i // 16]), :, i % 16] = 1000.0
    got = t.cache.attention(q.cuda(), t.batch)
    t.k, t.v = t.cache.k.cpu(), t.cache.v.cpu()
    for row, s, at in t.each_row():
        k, v = (torch.cat((oracle.keys_of(x, t.prefix, 16, 40), oracle.keys_of(x, t.tables[s], 16, at + 1))) for x in (t.k, t.v))
        keep = torch.isfinite(k.float()).all(-1).all(-1)
        want, size, score = oracle.attention(q[row], k[keep], v[keep], 1 / math.sqrt(128))
        within(got[row], want, oracle.attention_bound(want, size, score, 128, len(k), act, cache))


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, BF16), (F16, F16)])
def test_a_few_large_weights_among_many_small_ones(act, cache):
    """One key far above twelve thousand others, which together weigh as much."""
    t = Setup([1], [9000], 1, 64, 16, cache, prefix=3001, seed=6)
    q = torch.zeros(1, 1, 64, dtype=act)
    q[0, 0, 0] = 1.0
    t.k[..., 0] = 0.0
    t.k[int(t.tables[0, 100]), 0, 5, 0] = 9.5
    t.cache.k.copy_(t.k)
    check_attention(t, q, 1, 1, 64, act, cache, scale=1.0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows,prefix", [(64, 1, 0), (128, 3, 100), (64, 40, 0), (128, 40, 100), (256, 1, 0)])
def test_small_weights_keep_their_bits(act, cache, hd, rows, prefix):
    """A key 16 above all others whose values are zero: the result is made of weights of 1.1e-7."""
    t = Setup([rows], [1000], 1, hd, 16, cache, prefix=prefix, seed=24)
    q = torch.zeros(rows, 2, hd, dtype=act)
    q[:, :, 0] = 1.0
    t.k[..., 0] = 0.0
    t.v.abs_()
    t.k[int(t.tables[0, 100 // 16]), 0, 100 % 16, 0] = 16.0
    t.v[int(t.tables[0, 100 // 16]), 0, 100 % 16] = 0.0
    t.cache.k.copy_(t.k)
    t.cache.v.copy_(t.v)
    check_attention(t, q, 2, 1, hd, act, cache, scale=1.0)


@pytest.mark.parametrize("act,cache", [(F32, F16), (BF16, BF16)])
def test_strides_orders_and_outputs(act, cache):
    t = Setup([1, 3, 2], [40, 50, 5], 2, 64, 16, cache, prefix=30, pad=2, seed=7)
    plain = normal(t.tokens, 8, 64, dtype=act, seed=7).cuda()
    want = t.cache.attention(plain, t.batch)
    fused = torch.randn(t.tokens, 12 * 64 + 8, device="cuda").to(act)
    q = fused[:, 8: 8 + 8 * 64].unflatten(1, (8, 64))
    q.copy_(plain)
    assert torch.equal(t.cache.attention(q, t.batch), want)
    odd = torch.empty(t.tokens, 8 * 64 + 1, dtype=act, device="cuda")[:, 1:].unflatten(1, (8, 64))  # odd addresses
    odd.copy_(plain)
    assert torch.equal(t.cache.attention(odd, t.batch), want)
    turned = plain.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    assert torch.equal(t.cache.attention(turned, t.batch), want)
    columns = plain.transpose(1, 2).contiguous().transpose(1, 2)  # elements of a head apart
    assert torch.equal(t.cache.attention(columns, t.batch), want)
    for out in (torch.full((t.tokens, 8, 64), 7.0, dtype=act, device="cuda"), torch.full((t.tokens, 513), 7.0, dtype=act, device="cuda")[:, 1:].unflatten(1, (8, 64)),
                torch.full((8, t.tokens, 64), 7.0, dtype=act, device="cuda").transpose(0, 1)):
        assert t.cache.attention(plain, t.batch, out=out) is out
        assert torch.equal(out[:6], want[:6]) and bool((out[6:] == 7).all())
    wide = torch.full((3, 9), -5, dtype=torch.int32, device="cuda")[:, 2:]  # a table inside another
    tables = wide[:, : t.tables.shape[1]]
    tables.copy_(t.tables)
    again = PagedBatch(tables, t.batch.starts, t.batch.lengths, prefix=t.batch.prefix, prefix_length=30)
    assert torch.equal(t.cache.attention(plain, again), want)
    no_status()


def test_bad_pages_are_not_touched():
    """Ids that the cache does not have, and lengths that the table does not have, leave a status and nothing else."""
    t = Setup([1, 1], [40, 20], 1, 64, 16, F32, prefix=20, seed=8, extra_width=0)
    q = normal(2, 2, 64, seed=8)
    k, v = normal(2, 1, 64, seed=9), normal(2, 1, 64, seed=10)
    for bad in (-1, t.pages, 2 ** 31 - 1, -2 ** 31):
        tables = t.tables.clone()
        tables[0, 1] = bad
        batch = PagedBatch(tables.cuda(), t.batch.starts, t.batch.lengths, prefix=t.batch.prefix, prefix_length=20)
        got = t.cache.attention(q.cuda(), batch)
        assert device_status(0) == 96
        ks, vs = (torch.cat((oracle.keys_of(x, t.prefix, 16, 20), oracle.keys_of(x, t.tables[0], 16, 40)[torch.cat((torch.arange(16), torch.arange(32, 40)))])) for x in (t.k, t.v))
        want, size, score = oracle.attention(q[0], ks, vs, 1 / 8)
        within(got[0], want, oracle.attention_bound(want, size, score, 64, len(ks), F32, F32))
        tables = t.tables.clone()
        tables[0, 2] = bad
        batch = PagedBatch(tables.cuda(), t.batch.starts, t.batch.lengths)
        before = t.cache.k.clone()
        t.cache.append(None, k.cuda(), v.cuda(), batch)
        assert device_status(0) == 96
        changed = (t.cache.k.view(torch.int32) != before.view(torch.int32)).any(-1).any(1).nonzero().tolist()
        assert changed == [[int(t.tables[1, 19 // 16]), 19 % 16]]
        t.cache.k.copy_(before)
        prefix = t.prefix.clone()
        prefix[0] = bad
        got = t.cache.attention(q.cuda(), PagedBatch(t.tables.cuda(), t.batch.starts, t.batch.lengths, prefix=prefix.cuda(), prefix_length=20))
        assert device_status(0) == 96 and torch.isfinite(got).all()
    batch = PagedBatch(t.tables.cuda(), t.batch.starts, torch.tensor([2 ** 31 - 1, 20], dtype=torch.int32, device="cuda"))
    t.cache.append(None, k.cuda(), v.cuda(), batch)
    assert device_status(0) == 96
    batch = PagedBatch(t.tables.cuda(), t.batch.starts, torch.tensor([100, 20], dtype=torch.int32, device="cuda"))
    got = t.cache.attention(q.cuda(), batch)  # (the row sees what lies behind key 40 on its last page, where nothing finite is, and nothing of pages that are not in the table)
    assert device_status(0) == 96 and torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()
    for starts in ([0, 5, 9], [-3, 1, 2], [2, 1, 0], [7, 8, 9]):  # rows that are not there, or backwards
        batch = PagedBatch(t.tables.cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda"), t.batch.lengths, prefix=t.batch.prefix, prefix_length=20)
        assert torch.isfinite(t.cache.attention(q.cuda(), batch)).all()
        t.cache.append(q.cuda(), k.cuda(), v.cuda(), batch)
    device_status(0)


def test_pages_beyond_two_to_the_31_elements():
    """A cache of 2.3e9 elements, its sequences on the last pages."""
    pages, kv, hd, page = 17600, 8, 128, 128
    cache = PagedCache(pages, page, kv, hd, dtype=BF16)
    rope = Rope(1000, 128)
    freqs, magnitude = oracle.frequencies(128)
    tables = torch.tensor([[pages - 1, pages - 3], [pages - 2, 16500]], dtype=torch.int32, device="cuda")
    lengths = [150, 200]
    held = []
    for part in range(2):  # the lot at once, then one more row each
        rows = [149, 199] if part == 0 else [1, 1]
        starts = torch.tensor([0, rows[0], sum(rows)], dtype=torch.int32, device="cuda")
        batch = PagedBatch(tables, starts, torch.tensor([n - 1 + part for n in lengths], dtype=torch.int32, device="cuda"))
        q, k, v = (normal(sum(rows), h, hd, dtype=BF16, seed=s + part) for h, s in ((16, 20), (kv, 30), (kv, 40)))
        out = cache.attention(cache.append(q.cuda(), k.cuda(), v.cuda(), batch, rope=rope), batch)
        held.append((rows, q, k, v))
    for s in range(2):
        turned = lambda x, at: oracle.rotated(x, at, freqs, magnitude, False)[0].to(BF16)  # noqa: E731
        first = 0 if s == 0 else 149
        ks = torch.stack([turned(held[0][2][first + i], i) for i in range(lengths[s] - 1)] + [turned(held[1][2][s], lengths[s] - 1)])
        vs = torch.cat((held[0][3][first: first + lengths[s] - 1], held[1][3][s][None]))
        want, size, score = oracle.attention(turned(held[1][1][s], lengths[s] - 1), ks, vs, 1 / math.sqrt(hd))
        # queries and keys may be a step off where a rotation falls between two of their numbers: as a score, two half steps of each product
        within(out[s], want, oracle.attention_bound(want, size, score * (1 + 2 * 2.0 ** -8 * 2.0 ** 23 / (hd + 8) / 2), hd, len(ks), BF16, BF16))
    no_status()


def test_streams_and_graphs():
    """On another stream than the default, and captured: the replays read tables and lengths anew, and two graphs replayed at once have workspaces of their own."""
    t = Setup([1] * 6, [100, 7, 300, 31, 64, 1], 2, 128, 16, F16, prefix=200, seed=11)
    rope = Rope(1000, 128)
    q, k, v = (normal(6, h, 128, seed=s).cuda() for h, s in ((8, 1), (2, 2), (2, 3)))
    want = t.cache.attention(t.cache.append(q, k, v, t.batch, rope=rope), t.batch)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = t.cache.attention(t.cache.append(q, k, v, t.batch, rope=rope), t.batch)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs, batches = [], [], []
    for n in range(2):
        batch = PagedBatch(t.batch.tables.clone(), t.batch.starts.clone(), t.batch.lengths.clone(), prefix=t.batch.prefix, prefix_length=200)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = t.cache.attention(rope.rotate(q, 5), batch)
        graphs.append(g)
        outs.append(out)
        batches.append(batch)
    lengths = torch.tensor([3, 90, 12, 1, 0, 17], dtype=torch.int32)
    batches[1].lengths.copy_(lengths)
    torch.cuda.synchronize()
    plain = [t.cache.attention(rope.rotate(q, 5), b) for b in batches]
    for _ in range(20):
        for g, s in zip(graphs, (side, other)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    bits = [[x.view(torch.int32) for x in xs] for xs in (outs, plain)]  # (the other lengths reach what nobody has written: NaN)
    assert torch.equal(bits[0][0], bits[1][0]) and torch.equal(bits[0][1], bits[1][1]) and not torch.equal(bits[0][0], bits[0][1])
    no_status()


def test_the_same_bits_again():
    t = Setup([1, 5, 1, 2], [3000, 700, 1, 90], 2, 128, 16, F32, prefix=1500, seed=12)
    q = normal(t.tokens, 16, 128, seed=12).cuda()
    first = t.cache.attention(q, t.batch)
    for _ in range(5):
        assert torch.equal(t.cache.attention(q, t.batch), first)

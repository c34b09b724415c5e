"""Paged attention's numbers, by each of its kernels: infinities and NaN in values, keys and queries, weights far below the largest, and that rows of 32 bits keep them."""
import math

import pytest
import torch

import paged_oracle as oracle
from test_gpu_paged import TYPES, Setup, check_attention, no_status, normal, within

pytestmark = pytest.mark.gpu

# head size, rows and lengths of the sequences, prefix: the stream kernel, heads of 256 and of other sizes, and the tile kernel (where pages have 16 bits) for own keys, with a prefix, and for a
# prefix alone
SHAPES = [(64, [1, 3], [150, 90], 40), (128, [2], [300], 0), (256, [1, 2], [100, 70], 20), (40, [2, 1], [90, 40], 20), (64, [70, 2], [400, 30], 0), (128, [40, 9], [300, 290], 0),
          (128, [40], [200], 300), (64, [4] * 8, [60] * 8, 8200)]


def rows_of(t, q, hd):
    """Each row's keys' and values' places, and its result, weighted magnitudes and largest score in 64 bits, from the pages as they are."""
    k, v = t.cache.k.cpu(), t.cache.v.cpu()
    ahead = t.prefix_length
    for row, s, at in t.each_row():
        ks, vs = (torch.cat((oracle.keys_of(x, t.prefix, t.page, ahead) if ahead else x[:0, :, 0], oracle.keys_of(x, t.tables[s], t.page, at + 1))) for x in (k, v))
        yield row, ks, vs


def check_classes(t, q, kv, hd, act, cache):
    """Infinite and NaN elements of the values as the formula has them (the weights are above zero), all others within the bound."""
    got = t.cache.attention(q.cuda(), t.batch).cpu()
    odd = 0
    for row, k, v in rows_of(t, q, hd):
        group = q.shape[1] // kv
        finite = torch.isfinite(v.float())
        clean = torch.where(finite, v.float(), torch.zeros(()))
        want, size, score = oracle.attention(q[row], k, clean, 1 / math.sqrt(hd))
        bad = torch.where(finite, torch.zeros(()), v.float()).sum(0)  # [kv heads, head size]: infinity + -infinity is NaN
        bad = torch.where(finite.all(0), torch.zeros(()), bad).repeat_interleave(group, 0)
        plain = (bad == 0)
        bound = oracle.attention_bound(want, size, score, hd, len(k), act, cache)
        within(torch.where(plain, got[row].float(), torch.zeros(())), torch.where(plain, want, torch.zeros((), dtype=torch.float64)), bound, "row %d" % row)
        assert torch.equal(torch.isnan(got[row]), torch.isnan(bad)), "row %d" % row
        assert torch.equal(got[row].float()[torch.isinf(bad)], bad[torch.isinf(bad)]), "row %d" % row
        odd += int((~plain).sum())
    no_status()
    return odd


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows,lengths,prefix", SHAPES)
@pytest.mark.parametrize("place", ["first", "middle", "newest"])
def test_infinite_values_are_what_the_formula_says(act, cache, hd, rows, lengths, prefix, place):
    """Some elements of the values of a key are infinite or NaN, in the first run of keys, in the middle and (for those who see it) at the end."""
    t = Setup(rows, lengths, 2, hd, 16, cache, prefix=prefix, seed=41)
    q = normal(t.tokens, 8 if t.tokens > 8 else 4, hd, dtype=act, seed=41)
    own = {"first": 2, "middle": lengths[0] // 2 - 1, "newest": lengths[0] - 1}[place]
    places = [(t.tables[0], own)] + ([(t.prefix, {"first": 3, "middle": prefix // 2, "newest": prefix - 1}[place])] if prefix else [])
    for table, i in places:
        page, slot = int(table[i // 16]), i % 16
        t.cache.v[page, 0, slot, 1], t.cache.v[page, 0, slot, hd - 2], t.cache.v[page, 1, slot, 9] = math.inf, -math.inf, math.nan
    i = lengths[0] // 2  # another key of the same sequence: once the same infinity, once the other one
    page, slot = int(t.tables[0, i // 16]), i % 16
    t.cache.v[page, 0, slot, 1], t.cache.v[page, 0, slot, hd - 2] = math.inf, math.inf
    assert check_classes(t, q, 2, hd, act, cache) > 0


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows", [(64, 1), (128, 2), (64, 70), (128, 40)])
def test_an_infinite_value_alone(act, cache, hd, rows):
    """Its key has all the weight, one, whose smaller parts are zero. (One to a rounding: the score's product with log2(e) may be rounded once where the maximum is made and not where it is taken
    off, and as parts the weight has 22 bits in the products and 24 in the sum, so that the finite elements are the values to within attention_bound, whose docstring counts these.)"""
    t = Setup([rows], [200], 1, hd, 16, cache, seed=42)
    q = torch.zeros(rows, 2, hd, dtype=act)
    q[:, :, 0] = 8.0
    t.cache.k[..., 0] = 0.0
    page, slot = int(t.tables[0, 3]), 5
    t.cache.k[page, 0, slot, 0] = 500.0  # times 8 over at most 12: e^-333 for the others
    t.cache.v[page, 0, slot, 7], t.cache.v[page, 0, slot, 8] = math.inf, -math.inf
    assert check_classes(t, q, 1, hd, act, cache) == rows * 2 * 2


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows,prefix", [(64, [1], 0), (64, [70], 0), (128, [40], 0), (128, [40], 300), (64, [4] * 8, 8200), (128, [2] * 16, 4100)])
@pytest.mark.parametrize("far", [16, 18, 20, 21])
def test_weights_of_keys_far_below_the_largest(act, cache, hd, rows, prefix, far):
    """A key that far above all others, whose value is zero: the result is made of weights down to 7.6e-10, by each kernel."""
    t = Setup(rows, [max(900, n) for n in rows] if len(rows) == 1 else rows, 1, hd, 16, cache, prefix=prefix, seed=43)
    heads = 2 if len(rows) == 1 else 32
    q = torch.zeros(t.tokens, heads, hd, dtype=act)
    q[:, :, 0] = 1.0
    t.k[..., 0] = 0.0
    t.v.abs_()
    page, slot = (int(t.prefix[5]), 3) if prefix else (int(t.tables[0, 5]), 3)
    t.k[page, 0, slot, 0] = float(far)
    t.v[page, 0, slot] = 0.0
    t.v.mul_(1000.0)  # (so that results are among the type's ordinary numbers)
    t.cache.k.copy_(t.k)
    t.cache.v.copy_(t.v)
    check_attention(t, q, heads, 1, hd, act, cache, scale=1.0)


def check_scores(t, q, kv, hd, act, cache):
    """Keys that are not finite, as the formula has them: a score of minus infinity weighs nothing, one of infinity or NaN makes its row NaN; rows that do not see the key are what they were."""
    got = t.cache.attention(q.cuda(), t.batch).cpu()
    kinds = set()
    for row, k, v in rows_of(t, q, hd):
        heads, group = q.shape[1], q.shape[1] // kv
        for h in range(heads):
            keys = k[:, h // group].double()
            s = (keys * q[row, h].double()).sum(-1) / math.sqrt(hd)
            plain = torch.isfinite(keys).all(-1)
            if torch.isnan(s).any() or (s == math.inf).any():
                assert torch.isnan(got[row, h]).all(), "row %d, head %d" % (row, h)
                kinds.add("nan")
                continue
            assert (s[~plain] == -math.inf).all()
            kinds.add("zero" if not plain.all() else "plain")
            want, size, score = oracle.attention(q[row, h: h + 1], k[plain][:, h // group: h // group + 1], v[plain][:, h // group: h // group + 1], 1 / math.sqrt(hd))
            within(got[row, h: h + 1], want, oracle.attention_bound(want, size, score, hd, len(k), act, cache), "row %d, head %d" % (row, h))
    no_status()
    return kinds


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows,lengths,prefix", SHAPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("place", ["first", "newest"])
def test_keys_that_are_not_finite(act, cache, hd, rows, lengths, prefix, bad, place):
    """One element of a key: infinite scores have the sign of the query's element. Another key is minus infinity all over for one head, whose queries are positive."""
    t = Setup(rows, lengths, 2, hd, 16, cache, prefix=prefix, seed=44)
    q = normal(t.tokens, 8 if t.tokens > 8 else 4, hd, dtype=act, seed=44)
    group = q.shape[1] // 2
    q[:, :group] = q[:, :group].abs() + 0.25
    own = 1 if place == "first" else lengths[0] - 1
    t.cache.k[int(t.tables[0, own // 16]), 1, own % 16, 5] = bad
    own = 2 if place == "first" else lengths[0] - 1
    t.cache.k[int(t.tables[0, own // 16]), 0, own % 16] = -math.inf
    kinds = check_scores(t, q, 2, hd, act, cache)
    assert "zero" in kinds and ("nan" in kinds or (t.tokens < 9 and bad == bad))  # (few queries may all have the sign that makes minus infinity)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hd,rows,lengths,prefix", SHAPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite(act, cache, hd, rows, lengths, prefix, bad):
    """An element of one row's queries, or all of them: that row is NaN, the others are what they were to the bit."""
    t = Setup(rows, lengths, 2, hd, 16, cache, prefix=prefix, seed=45)
    q = normal(t.tokens, 8 if t.tokens > 8 else 4, hd, dtype=act, seed=45).cuda()
    clean = t.cache.attention(q, t.batch)
    row, other = 0, t.starts[1] - 1
    q[row, 0], q[other, -1, 3] = bad, bad
    got = t.cache.attention(q, t.batch)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    hit[row, 0] = hit[other, -1] = True
    assert torch.isnan(got[hit]).all()
    bits = torch.int32 if act is torch.float32 else torch.int16
    assert torch.equal(got[~hit].view(bits), clean[~hit].view(bits))
    no_status()


@pytest.mark.parametrize("cache", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd,rows,lengths,prefix", SHAPES + [(128, [1], [577], 0), (64, [200], [1100], 0), (128, [100], [600], 900)])
def test_rows_of_32_bits_keep_them(cache, hd, rows, lengths, prefix):
    """The root mean square of the error is at most 1e-6 of the results'. A weight is off by up to 2^-22 of itself as parts of 22 bits, by 2^-22 for its exponential, and by its score's error: hd
    products exact to 2^-22 with random signs, 2^-22 of their root of squares, which is about 1 for normal numbers; sums and the quotient are rounded to 2^-24. Errors of different keys have no common
    sign, so that of the result they make at most 2^-22 (1 + 1 + 1 + 1/2) = 8.3e-7. (Queries and keys as one half-precision number each, 3.3e-4, or queries as one bfloat16 number,
    1.6e-3, are within attention_bound for many of these shapes.)"""
    t = Setup(rows, lengths, 2, hd, 16, cache, prefix=prefix, seed=46)
    q = normal(t.tokens, 8 if t.tokens > 8 else 4, hd, seed=46)
    got = t.cache.attention(q.cuda(), t.batch).cpu().double()
    off = size = 0.0
    for row, k, v in rows_of(t, q, hd):
        want = oracle.attention(q[row], k, v, 1 / math.sqrt(hd))[0]
        off += float(((got[row] - want) ** 2).sum())
        size += float((want ** 2).sum())
    assert math.sqrt(off / size) <= 1e-6, math.sqrt(off / size)
    no_status()

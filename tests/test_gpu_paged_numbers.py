"""Paged attention where numbers are not ordinary: infinities and NaN that a row sees or does not, by each of its kernels."""
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

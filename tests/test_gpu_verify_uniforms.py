"""Verification where the uniform numbers lie outside [0, 1), or on the borders between the pieces that the kernel cuts a row's weights into: every token is one that has a weight."""
import math

import pytest
import torch

import paged_oracle as oracle
from jitnn_b200 import Speculative
from test_gpu_verify import case

pytestmark = pytest.mark.gpu


def verify(c):
    return [x.tolist() for x in Speculative.verify(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()})]


@pytest.mark.parametrize("temperature", [None, 0.8])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("vocab", [3, 100, 5000, 40000])
def test_negative_uniforms_count_as_zero(temperature, drafter, vocab):
    c = case(6, 3, vocab, torch.float32, temperature, drafter, False, seed=11)
    c["target"][:, :, 0] = 0.0 if temperature is None else -math.inf  # (the first token has no weight)
    c["drafts"][3:] = 0
    zero = torch.zeros_like(c["uniforms"])
    want = list(oracle.verify(c["target"], c["drafts"], zero, c.get("draft_probs"), None, temperature))
    for u in (0.0, -0.0, -1e-40, -0.3, -1.0, -3e38, -math.inf):
        c["uniforms"] = torch.full_like(zero, u)
        assert verify(c) == want, u
    assert all(t[a] != 0 for a, t in zip(*want))


@pytest.mark.parametrize("vocab", [4096, 60000, 131072])
def test_borders_between_the_pieces(vocab):
    """Weights that no sum holds exactly, whole runs of the row without any, aims at each run's border and a step beside it."""
    g = torch.Generator().manual_seed(12)
    run = vocab // 128
    keep = torch.rand(128, generator=g) < 0.3
    keep[5] = True
    p = torch.rand(vocab, generator=g) * keep.repeat_interleave(run)[:vocab] if vocab % 128 == 0 else torch.rand(vocab, generator=g) * torch.cat((keep.repeat_interleave(run), keep[-1:].repeat(vocab - 128 * run)))
    p = p / p.sum()
    upto = p.double().cumsum(0)
    u = (upto[run - 1:: run] / upto[-1]).float()
    u = torch.cat((u, torch.nextafter(u, torch.zeros(())), torch.nextafter(u, torch.ones(())))).clamp(0, 1)
    _, tokens = Speculative.verify(p.cuda().expand(len(u), 1, vocab), torch.zeros(len(u), 0, dtype=torch.int32, device="cuda"), u[:, None].cuda())
    tokens = tokens[:, 0].long().cpu()
    assert ((0 <= tokens) & (tokens < vocab)).all() and (p[tokens] > 0).all()
    # the token's interval has the aim to within the rounding of sums of at most `vocab` terms that add up to one, each vocab 2^-53: the aim's total and the border, here and there
    aim, slack = u.double() * upto[-1], 4 * vocab * 2.0 ** -53
    assert (aim < upto[tokens] + slack).all()
    assert (aim >= upto[tokens] - p[tokens].double() - slack).all()

"""Verification of drafted tokens against a plain 64-bit form: whole numbers, equal ones."""
import math

import pytest
import torch

import paged_oracle as oracle
from jitnn_b200 import Speculative, device_status

pytestmark = pytest.mark.gpu


def case(sequences, drafts, vocab, dtype, temperature, drafter, ragged, seed=0, size=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(sequences, drafts + 1, vocab, generator=g) * size
    target = torch.softmax(logits, -1) if temperature is None else logits.to(dtype)
    noise = logits[:, :drafts] + torch.randn(sequences, drafts, vocab, generator=g)
    q = torch.softmax(noise / (temperature or 1.0), -1)
    x = torch.multinomial(q.reshape(-1, vocab), 1, generator=g).reshape(sequences, drafts).int() if drafts else torch.zeros(sequences, 0, dtype=torch.int32)
    if not drafter or temperature == 0:
        x = torch.where(torch.rand(x.shape, generator=g) < 0.7, logits[:, :drafts].argmax(-1).int(), x)
    return {"target": target, "drafts": x, "uniforms": torch.rand(sequences, drafts + 1, generator=g), "draft_probs": q if drafter else None,
            "counts": torch.randint(0, drafts + 1, (sequences,), generator=g).int() if ragged else None, "temperature": temperature}


def check(c):
    accepted, tokens = Speculative.verify(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()})
    assert accepted.dtype is torch.int32 and tokens.dtype is torch.int32
    want = oracle.verify(**c)
    assert accepted.tolist() == want[0] and tokens.tolist() == want[1]
    return accepted.tolist(), tokens.tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temperature", [None, 0.0, 0.4, 1.0, 7.0])
@pytest.mark.parametrize("sequences,drafts,vocab", [(1, 1, 1), (1, 4, 7), (5, 3, 1000), (3, 8, 32001), (70, 2, 513), (2, 0, 4097), (1, 5, 131071), (9, 7, 8192)])
@pytest.mark.parametrize("drafter,ragged", [(True, False), (False, True)])
def test_verify(dtype, temperature, sequences, drafts, vocab, drafter, ragged):
    c = case(sequences, drafts, vocab, dtype, temperature, drafter, ragged, seed=sequences + drafts)
    check(c)
    assert device_status(0) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-300, 1e-40, 1e-20, 1e-9, 1e-7, 1e-5, 1e4, 1e30])
@pytest.mark.parametrize("size", [1e-3, 3.0, 1e4, 1e10, 1e30])
def test_logits_and_temperatures_of_any_size(dtype, temperature, size):
    """From all but one weight zero to all weights the same; logits whose steps are far above the temperature, equal ones and masked ones (minus infinity) among them."""
    c = case(4, 3, 5003, dtype, 1.0, False, False, seed=11, size=size)
    c["temperature"] = temperature
    c["target"][0, :, ::7] = c["target"][0].amax(-1, keepdim=True)
    c["target"][1, :, 100:] = -math.inf
    c["drafts"][2] = c["target"][2, :3].argmax(-1).int()
    check(c)
    assert device_status(0) == 0


def test_each_way_out():
    """All kept, none kept, refused in between; the drafter's own distribution: p and q are the same, the token comes from p."""
    c = case(64, 4, 50, torch.float32, None, True, False, seed=1, size=1.0)
    accepted, _ = check(c)
    assert set(accepted) >= {0, 2, 4}
    c["draft_probs"] = c["target"][:, :4].clone()  # u < 1: everything with a probability is kept
    assert set(check(c)[0]) == {4}
    c["uniforms"][:, :4] = 0.0
    c["draft_probs"].mul_(0.0)
    check(c)


def test_a_refused_draft_and_no_weight_left():
    """q above p everywhere (it is no distribution): the token comes from p."""
    target = torch.tensor([[[0.25, 0.25, 0.5], [0.2, 0.3, 0.5]]])
    q = torch.full((1, 1, 3), 2.0)
    for u in (0.0, 0.3, 0.9):
        c = {"target": target, "drafts": torch.tensor([[1]], dtype=torch.int32), "uniforms": torch.tensor([[0.9, u]]), "draft_probs": q}
        assert check(c)[0] == [0]


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24])
def test_borders(u):
    """Equal weights that sums hold exactly: an aim on a border goes to the token behind it; tokens without weight are never drawn."""
    p = torch.zeros(1, 1, 4096)
    p[0, 0, 5::8] = 2.0 ** -9
    c = {"target": p, "drafts": torch.zeros(1, 0, dtype=torch.int32), "uniforms": torch.tensor([[u]])}
    token = check(c)[1][0][0]
    assert token % 8 == 5 and token == 5 + 8 * min(511, math.floor(u * 512))


def test_masked_logits_and_equal_maxima():
    c = case(3, 2, 3000, torch.float32, 1.0, False, False, seed=2)
    c["target"][:, :, ::2] = -math.inf  # tokens that are not allowed
    check(c)
    c["target"][1] = -math.inf
    c["target"][1, :, 1234] = 5.0  # one token alone
    c["drafts"][1] = 1234
    assert check(c)[1][1] == [1234] * 3
    c["temperature"], c["uniforms"] = 0.0, None
    c["target"][0] = 1.5  # all the same: the first
    check(c)
    c["target"][2, :, 77] = c["target"][2, :, 2999] = 100.0
    c["target"][2, :, 76] = c["target"][2, :, 2998] = math.nan  # never the likeliest
    c["drafts"][2] = 77
    accepted, tokens = Speculative.verify(c["target"].cuda(), c["drafts"].cuda(), temperature=0.0)
    assert tokens[2].tolist() == [77, 77, 77] and tokens[0, int(accepted[0])] == 0


def test_large_logits_and_low_temperatures():
    c = case(4, 3, 2000, torch.float32, 0.01, False, False, seed=3)
    check(c)
    c["target"].mul_(1000.0)
    check(c)
    c["target"] += 1e30
    check(c)


def test_numbers_that_should_not_be_there():
    """Drafts outside the vocabulary are refused and leave a status; uniforms of one and more, or none, give the last token with any weight; nothing is read out of range."""
    c = case(4, 2, 100, torch.float32, 1.0, False, False, seed=4)
    c["drafts"][0, 0], c["drafts"][1, 1], c["drafts"][2, 0] = 100, -1, 2 ** 31 - 1
    check(c)
    assert device_status(0) == 98
    p = torch.zeros(3, 1, 100)
    p[:, 0, 10:21] = 1 / 11
    u = torch.tensor([[1.0], [2.0], [math.nan]])
    _, tokens = Speculative.verify(p.cuda(), torch.zeros(3, 0, dtype=torch.int32, device="cuda"), u.cuda())
    assert tokens.tolist() == [[20]] * 3
    p[0] = math.nan
    p[1] = 0.0
    _, tokens = Speculative.verify(p.cuda(), torch.zeros(3, 0, dtype=torch.int32, device="cuda"), (u * 0 + 0.5).cuda())
    assert tokens.tolist()[:2] == [[99]] * 2
    c = case(3, 2, 100, torch.float32, 1.0, False, False, seed=5)
    want = check(c)
    c["counts"] = torch.tensor([5, 2 ** 31 - 1, 2], dtype=torch.int32)  # more than there are: all
    accepted, tokens = Speculative.verify(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()})
    assert (accepted.tolist(), tokens.tolist()) == want
    c["counts"] = torch.tensor([-7, 0, -2 ** 31], dtype=torch.int32)
    accepted, _ = Speculative.verify(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()})
    assert accepted.tolist() == [0, 0, 0]
    assert device_status(0) == 0


def test_strides_streams_and_graphs():
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in case(4, 3, 5000, torch.float32, 0.9, True, True, seed=6).items()}
    want = [x.tolist() for x in Speculative.verify(**c)]
    d = dict(c)
    wide = torch.randn(4, 5, 5003, device="cuda")
    wide[:, 1:, 2:5002] = c["target"]
    d["target"] = wide[:, 1:, 2:5002]
    d["draft_probs"] = torch.cat((c["draft_probs"], c["draft_probs"]), 2)[:, :, 5000:]
    d["uniforms"] = torch.stack((c["uniforms"], c["uniforms"]), -1)[..., 1]
    assert [x.tolist() for x in Speculative.verify(**d)] == want
    d["target"] = c["target"].transpose(1, 2).contiguous().transpose(1, 2)
    assert [x.tolist() for x in Speculative.verify(**d)] == want
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = Speculative.verify(**c)
    side.synchronize()
    assert [x.tolist() for x in got] == want
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = Speculative.verify(**c)
    c["target"].copy_(c["target"].flip(2))
    g.replay()
    torch.cuda.synchronize()
    assert [x.tolist() for x in got] == [x.tolist() for x in Speculative.verify(**c)]
    with pytest.raises(ValueError, match="uniforms"):
        Speculative.verify(c["target"], c["drafts"], None, temperature=1.0)
    empty = Speculative.verify(c["target"][:0], c["drafts"][:0], c["uniforms"][:0])
    assert empty[0].shape == (0,) and empty[1].shape == (0, 4)

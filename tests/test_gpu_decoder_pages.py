"""The decoder on paged caches against the CPU oracle of the reference's Llama block math: single tokens and runs, sequences of different lengths behind a shared prefix, drafts verified
against the logits, and a rescaled rotation on both kinds of caches. Logits with FP32 pages within 2e-4 of the largest magnitude, as the decoder's other paths."""
import numpy as np
import pytest
import torch

import paged_oracle
from jitnn_b200 import LlamaDecoder, RopeScaling
from oracle import llama_oracle

pytestmark = pytest.mark.gpu


def build(dim, heads, kv_heads, max_seq=200, scaling=None, seed=1, vocab=512):
    cfg = llama_oracle.Config(layers=2, dim=dim, heads=heads, kv_heads=kv_heads, hidden=2 * dim, vocab=vocab, max_seq=max_seq)
    weights = llama_oracle.random_model(cfg, seed)
    dec = LlamaDecoder(cfg.layers, cfg.dim, cfg.heads, cfg.kv_heads, cfg.hidden, cfg.vocab, cfg.max_seq, cfg.eps, cfg.rope_base, rope_scaling=scaling)
    dec.load(weights)
    return cfg, weights, dec


def reference(cfg, weights, tokens):
    ref = llama_oracle.Decoder(cfg, weights)
    return np.stack([ref.forward(int(t), i) for i, t in enumerate(tokens)])


def close(got, want, rel=2e-4):
    assert np.abs(got - want).max() <= rel * np.abs(want).max(), float(np.abs(got - want).max() / np.abs(want).max())


@pytest.mark.parametrize("dim,heads,kv_heads", [(256, 4, 2), (512, 4, 1), (512, 2, 2), (256, 8, 4), (512, 8, 1)])
def test_runs_and_single_tokens(dim, heads, kv_heads):
    """Head sizes 64, 128, 256 and (on the general kernel) 32."""
    cfg, weights, dec = build(dim, heads, kv_heads)
    dec.set_pages(20, 16, "F32")
    tokens = np.random.default_rng(2).integers(0, cfg.vocab, 50).astype(np.int32)
    want = reference(cfg, weights, tokens)
    table, at = [7, 3, 19, 0], 0
    for n in (1, 16, 1, 5, 16, 1, 1, 9):
        logits, nxt = dec.forward_pages([tokens[at: at + n]], [table], [at + n])
        close(logits, want[at: at + n])
        assert nxt.tolist() == logits.argmax(-1).tolist()
        at += n
    assert at == 50
    # the contiguous caches are where they were
    close(dec.forward(tokens[:8], 0)[0], want[:8])
    close(dec.forward_pages([tokens[49:50]], [table], [50])[0], want[49:])  # the same keys again


@pytest.mark.parametrize("dtype,rel", [("F32", 2e-4), ("F16", 5e-3), ("BF16", 4e-2)])
@pytest.mark.parametrize("dim,heads,kv_heads", [(512, 4, 1), (256, 4, 4)])
def test_sequences_behind_a_prefix(dtype, rel, dim, heads, kv_heads):
    """A prefix of 37 tokens once, then three sequences of their own lengths, one of which sits a step out. Keys and values of 16 bits are up to half a step, 2^-11 or 2^-8,
    off, which two layers with their residual sums and norms carry on to the logits: ten times that."""
    cfg, weights, dec = build(dim, heads, kv_heads, seed=3)
    dec.set_pages(40, 16, dtype)
    rng = np.random.default_rng(4)
    prefix = rng.integers(0, cfg.vocab, 37)
    pages = list(rng.permutation(40))
    ahead, tables = pages[:3], [pages[3:6], pages[6:9], pages[9:12]]
    for at in range(0, 37, 16):  # the prefix as a sequence of its own
        dec.forward_pages([prefix[at: at + 16]], [ahead], [min(37, at + 16)], want_logits=False)
    own = [list(rng.integers(0, cfg.vocab, n)) for n in (30, 9, 41)]
    want = [reference(cfg, weights, list(prefix) + t)[37:] for t in own]
    at = [0, 0, 0]
    for step in ([5, 3, 8], [1, 0, 1], [4, 1, 11], [1, 1, 1], [14, 0, 2], [1, 4, 10], [4, 0, 8]):
        tokens = [t[a: a + n] for t, a, n in zip(own, at, step)]
        at = [a + n for a, n in zip(at, step)]
        logits, _ = dec.forward_pages(tokens, tables, at, prefix=ahead, prefix_length=37)
        row = 0
        for w, a, n in zip(want, at, step):
            if n:
                close(logits[row: row + n], w[a - n: a], rel)
            row += n
    assert at == [30, 9, 41]


def test_drafts():
    """Greedy: drafts are kept as long as they are what the decoder would have said. At a temperature: the verification of the logits that forward_pages gives for the same tokens."""
    cfg, weights, dec = build(256, 4, 2, seed=5, vocab=300)
    dec.set_pages(16, 16, "F32")
    rng = np.random.default_rng(6)
    prompts = [list(rng.integers(0, cfg.vocab, n)) for n in (7, 11)]
    tables = [[2, 5], [9, 4]]
    first = []
    for p, t in zip(prompts, tables):
        first.append(int(dec.forward_pages([p], [t], [len(p)])[1][-1]))
    plain = []  # what comes without drafts
    for p, t, x in zip(prompts, tables, first):
        said = [x]
        for i in range(4):
            said.append(int(dec.forward_pages([[said[-1]]], [t], [len(p) + 1 + i])[1][0]))
        plain.append(said)
    tokens = np.array([[s[0], s[1], s[2], s[3]] for s in plain], dtype=np.int32)
    tokens[1, 2] = (tokens[1, 2] + 1) % cfg.vocab  # the second sequence's second draft is another
    lengths = [len(p) + 4 for p in prompts]
    accepted, got = dec.verify_pages(tokens, tables, lengths)
    assert accepted.tolist() == [3, 1]
    assert got.tolist() == [plain[0][1:5], [plain[1][1], plain[1][2], -1, -1]]
    # drafts refused: the next call goes on behind what was kept
    logits, nxt = dec.forward_pages([[plain[1][2]]], [tables[1]], [len(prompts[1]) + 3])
    close(logits, reference(cfg, weights, prompts[1] + plain[1][:3])[-1:])
    logits, _ = dec.forward_pages(list(tokens), tables, lengths)
    uniforms = rng.random((2, 4), dtype=np.float32)
    q = rng.random((2, 3, cfg.vocab), dtype=np.float32)
    q /= q.sum(-1, keepdims=True)
    for probs in (None, q):
        for temperature in (0.7, 3.0):
            accepted, got = dec.verify_pages(tokens, tables, lengths, uniforms, probs, temperature)
            want = paged_oracle.verify(torch.from_numpy(logits).view(2, 4, -1), torch.from_numpy(tokens[:, 1:]), torch.from_numpy(uniforms), None if probs is None else torch.from_numpy(q),
                                       temperature=temperature)
            assert (accepted.tolist(), got.tolist()) == want
    accepted, got = dec.verify_pages(tokens[:, :1], tables, [n - 3 for n in lengths], uniforms[:, :1], temperature=1.0)  # no drafts: sampling
    assert accepted.tolist() == [0, 0] and ((0 <= got) & (got < cfg.vocab)).all()


@pytest.mark.parametrize("scaling,oracle_scaling", [(RopeScaling.linear(4), ("linear", 4.0)), (RopeScaling.llama3(8, 1, 4, 64), ("llama3", 8.0, 1.0, 4.0, 64.0)),
                                                    (RopeScaling.yarn(4, 64), ("yarn", 4.0, 64.0, 32.0, 1.0))])
def test_rescaled_rotation(scaling, oracle_scaling, monkeypatch):
    cfg, weights, dec = build(256, 4, 2, scaling=scaling, seed=7)
    freqs, magnitude = paged_oracle.frequencies(cfg.head_dim, cfg.rope_base, oracle_scaling)

    def tables(c):
        angle = np.arange(c.max_seq, dtype=np.float64)[:, None] * np.array(freqs)[None]
        return (np.cos(angle) * magnitude).astype(np.float32), (np.sin(angle) * magnitude).astype(np.float32)

    tokens = np.random.default_rng(8).integers(0, cfg.vocab, 40).astype(np.int32)
    unscaled = reference(cfg, weights, tokens)
    monkeypatch.setattr(llama_oracle, "rope_tables", tables)
    want = reference(cfg, weights, tokens)
    assert np.abs(want - unscaled).max() > 1e-2 * np.abs(want).max()
    close(np.concatenate([dec.forward(tokens[i: i + 8], i)[0] for i in range(0, 40, 8)]), want)
    close(np.stack([dec.forward(tokens[i: i + 1], i, seq=0)[0][0] for i in range(40)]), want)
    dec.set_pages(8, 16, "F32")
    close(np.concatenate([dec.forward_pages([tokens[i: i + 8]], [[1, 6, 3]], [i + 8])[0] for i in range(0, 40, 8)]), want)


def test_refusals():
    cfg, _, dec = build(256, 4, 2)
    with pytest.raises(ValueError, match="no pages"):
        dec.forward_pages([[1]], [[0]], [1])
    for bad in (15, 24, 2048, 0):
        with pytest.raises(ValueError, match="power of two"):
            dec.set_pages(4, bad)
    with pytest.raises(ValueError, match="pages of type"):
        dec.set_pages(4, 16, "Q8_0")
    dec.set_pages(4, 16, "F16")
    for args, message in ((([[1]], [[4]], [1]), "has page 4 of 4"), (([[1]], [[-1]], [1]), "has page -1"), (([[1]], [[0]], [17]), "17 keys on 1 pages"), (([[1, 2]], [[0]], [1]), "2 new tokens, 1 keys"),
                          (([[1] * 17], [[0, 1]], [17]), "17 new tokens"), (([[1] * 9, [2] * 8], [[0], [1]], [9, 8]), "17 tokens"), (([[]], [[0]], [1]), "0 tokens"),
                          (([[1]], [[0]] * 2, [1, 2]), "1 sequences, 2 lengths"), (([[1]], [list(range(4)) * 4], [201]), "201 keys behind a prefix of 0")):
        with pytest.raises(ValueError, match=message):
            dec.forward_pages(*args)
    for prefix, length, message in (([9], 5, "the prefix has page 9"), ([1], 17, "17 keys on 1 pages"), (None, 3, "3 keys on 0 pages"), ([1], -1, "-1 keys"), ([0, 1, 2, 3] * 4, 200, "behind a prefix of 200")):
        with pytest.raises(ValueError, match=message):
            dec.forward_pages([[1]], [[0]], [1], prefix=prefix, prefix_length=length)
    with pytest.raises(ValueError, match="temperature"):
        dec.verify_pages([[1, 2]], [[0]], [2], temperature=1.0)
    with pytest.raises(ValueError, match="temperature -1"):
        dec.verify_pages([[1, 2]], [[0]], [2], temperature=-1.0)
    with pytest.raises(ValueError, match="temperature 1e"):
        dec.verify_pages([[1, 2]], [[0]], [2], uniforms=[[0.5, 0.5]], temperature=1e31)
    with pytest.raises(ValueError, match="uniforms of shape"):
        dec.verify_pages([[1, 2]], [[0]], [2], uniforms=[[0.5]], temperature=1.0)
    with pytest.raises(ValueError, match="outside the vocabulary"):
        dec.verify_pages([[1, 512]], [[0]], [2])
    dec.forward_pages([[1]], [[0]], [1])
    dec.set_pages(0)
    with pytest.raises(ValueError, match="no pages"):
        dec.forward_pages([[1]], [[0]], [1])

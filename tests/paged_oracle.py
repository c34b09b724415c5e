"""Plain 64-bit forms of the operators of paged decoding, on the CPU, one row at a time, and how far a kernel may be from them."""
import math

import torch

# elements and half a step of each type
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step among the smallest numbers


def frequencies(dim, base=10000.0, scaling=None):
    """scaling: None or (kind, parameters ...). Pair after pair from the definitions."""
    got, magnitude = [], 1.0
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        if scaling is not None and scaling[0] == "linear":
            f /= scaling[1]
        elif scaling is not None and scaling[0] == "llama3":
            _, factor, low, high, context = scaling
            turns = context * f / (2 * math.pi)
            if turns < low:
                f /= factor
            elif turns <= high:
                part = (turns - low) / (high - low)
                f = part * f + (1 - part) * f / factor
        elif scaling is not None:
            _, factor, context, fast, slow = scaling
            magnitude = 0.1 * math.log(factor) + 1
            edge = [dim * math.log(context / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow)]
            first, last = max(0, math.floor(edge[0])), min(dim - 1, math.ceil(edge[1]))
            part = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = (1 - part) * f + part * f / factor
        got.append(f)
    return got, magnitude


def rotated(x, position, freqs, magnitude, interleaved, back=False):
    """x [heads, head size] in 64 bits, and what its absolute values give (the scale of the rounding errors)."""
    x = x.double()
    n = len(freqs)
    a = torch.tensor([position * f * (-1 if back else 1) for f in freqs], dtype=torch.float64)
    c, s = a.cos() * magnitude, a.sin() * magnitude
    i = (torch.arange(n) * 2, torch.arange(n) * 2 + 1) if interleaved else (torch.arange(n), torch.arange(n) + n)
    y, size = x.clone(), torch.zeros_like(x)
    u, v = x[:, i[0]], x[:, i[1]]
    y[:, i[0]], y[:, i[1]] = u * c - v * s, u * s + v * c
    size[:, i[0]], size[:, i[1]] = (u * c).abs() + (v * s).abs(), (u * s).abs() + (v * c).abs()
    return y, size


def rotation_bound(y, size, dtype):
    """Cosine, product and sum are each rounded to 24 bits: three half steps of each product, one of the sum (at most the products' size); then the result to its type."""
    return 4 * 2.0 ** -24 * size + HALF_STEP[dtype] * (y.abs() + 4 * 2.0 ** -24 * size) + SMALLEST[dtype]


def keys_of(pages, table, page_size, count):
    """[count, heads, head size] of a cache [pages, heads, page size, head size]."""
    i = torch.arange(count)
    return pages[table[i // page_size].long(), :, i % page_size]


def attention(q, k, v, scale):
    """q [heads, head size] over k, v [keys, kv heads, head size]: (out, weighted magnitudes, magnitude of the largest score's sum), 64 bits."""
    group = q.shape[0] // k.shape[1]
    k, v = k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    q = q.double()
    s = torch.einsum("hd,jhd->hj", q, k) * scale
    p = torch.softmax(s, -1)
    return torch.einsum("hj,jhd->hd", p, v), torch.einsum("hj,jhd->hd", p, v.abs()), torch.einsum("hd,jhd->hj", q.abs(), k.abs()).amax(-1) * abs(scale)


def attention_bound(out, size, score, head_dim, keys, act, cache):
    """How far a row may be off. A score is a sum of head_dim products whose factors are exact to 2^-22 (FP32 rows may be held as sums of shorter numbers), added up in
    32 bits in any order, times the scale and log2(e): off by at most (head_dim + 8) 2^-23 of the sum of magnitudes. A weight e^(s - m) is off by that, twice (m has the
    same error), by 2^-21 of its own (the exponential, and parts of 22 bits) and, where rows have 16 bits, by a rounding to the pages' type. Weighted values and weights
    are added up in 32 bits: sums of `keys` terms in runs of at most 4096 that are joined, (4096 + keys / 4096) 2^-24 in the worst case. Numerator and denominator each
    have these errors; the quotient is rounded to the rows' type."""
    weight = 2 * (head_dim + 8) * 2.0 ** -23 * score + 2.0 ** -21 + (0 if act is torch.float32 else HALF_STEP[cache]) + (min(keys, 4096) + keys / 4096 + 8) * 2.0 ** -24
    off = 2 * (torch.exp(weight) - 1)[:, None] * size
    return off + HALF_STEP[act] * (out.abs() + off) + SMALLEST[act]


def verify(target, drafts, uniforms, draft_probs=None, counts=None, temperature=None):
    """One sequence after the other; target [sequences, drafts + 1, vocab]. Lists."""
    accepted, tokens = [], []
    n, rows, vocab = target.shape
    for b in range(n):
        count = rows - 1 if counts is None else int(counts[b])
        got = []

        def row(i):
            x = target[b, i].double()
            return x if temperature is None else torch.softmax((x - x.max()) / temperature, -1)  # (1e10 / 1e-300 is above the largest double)

        def likeliest(i):
            x = target[b, i].double()
            return int((x == x.max()).nonzero()[0])

        while len(got) < count:
            i, x = len(got), int(drafts[b, len(got)])
            if not 0 <= x < vocab:
                break
            if temperature == 0:
                keep = x == likeliest(i)
            else:
                keep = float(uniforms[b, i]) * (1.0 if draft_probs is None else float(draft_probs[b, i, x])) < float(row(i)[x])
            if not keep:
                break
            got.append(x)
        j = len(got)
        if temperature == 0:
            token = likeliest(j)
        else:
            p = row(j)
            w = p.clone()
            if j < count:
                if draft_probs is not None:
                    w = w - draft_probs[b, j].double()
                elif 0 <= int(drafts[b, j]) < vocab:
                    w[int(drafts[b, j])] = 0
            w = torch.nan_to_num(w, nan=0.0).clamp(min=0)
            if float(w.sum()) == 0:
                w = torch.nan_to_num(p, nan=0.0).clamp(min=0)
            upto = w.cumsum(0)
            over = (upto > float(uniforms[b, -1]) * float(upto[-1])).nonzero()
            token = int(over[0]) if len(over) else vocab - 1
        accepted.append(j)
        tokens.append(got + [token] + [-1] * (rows - 1 - j))
    return accepted, tokens

"""The operators of paged decoding as cases that can be timed and compared: rotary positions, the append to a paged cache, attention over it for a batch
that shares a prefix, and the verification of drafted tokens.

A case is a dict of plain values. Its "kind" says which operator it stands for:

* ``rope``    ``Rope.rotate`` of queries and keys, or with "backward" ``Rope.backward`` of their gradients.
* ``append``  ``PagedCache.append``: the rotation of new queries and keys, and keys and values into their pages.
* ``attend``  ``PagedCache.attention``: each row over the shared prefix and its own sequence's keys.
* ``verify``  ``Speculative.verify``: drafted tokens against the target's logits or probabilities.

With ``own`` false ``run`` computes them from elementary torch operations, with ``own`` true through the library.
"""
import math

import torch

own = False

# heads, key/value heads, head size
HEADS = {"small": (16, 16, 64), "7b": (32, 32, 128), "7b-gqa": (32, 8, 128), "70b": (64, 8, 128), "gqa-64": (32, 8, 64), "wide": (16, 4, 256)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
POSITIONS = 32768  # of every table of rotations
BASE = 500000.0


def listed():
    return [
        # one new token of one sequence, full precision: the smallest call, latency counts
        {"name": "rope_step_f32", "kind": "rope", "heads": "7b", "batch": 1, "seq": 1, "type": "f32", "rot": 128, "interleaved": False, "scaling": "none", "backward": False},
        # a long prompt of a model whose context was stretched
        {"name": "rope_prompt_bf16", "kind": "rope", "heads": "70b", "batch": 1, "seq": 4096, "type": "bf16", "rot": 128, "interleaved": False, "scaling": "llama3", "backward": False},
        # the gradient for a small training batch of odd length, pairs next to each other in the first half of the head
        {"name": "rope_backward_f16", "kind": "rope", "heads": "7b-gqa", "batch": 3, "seq": 1365, "type": "f16", "rot": 64, "interleaved": True, "scaling": "yarn", "backward": True},
        # a decode step of sixteen sequences: one token each, a cache in half precision behind full-precision activations
        {"name": "append_step_f32_f16", "kind": "append", "heads": "70b", "sequences": 16, "rows": 1, "pad": 0, "type": "f32", "cache": "f16", "page": 16, "prefix": 1000, "most": 2048,
         "rot": 128, "interleaved": False, "scaling": "llama3"},
        # prompts of several sequences in one call, ragged, with rows of padding behind the last
        {"name": "append_prompts_bf16", "kind": "append", "heads": "7b-gqa", "sequences": 7, "rows": 1170, "pad": 2, "type": "bf16", "cache": "bf16", "page": 64, "prefix": 0, "most": 2400,
         "rot": 128, "interleaved": False, "scaling": "none"},
        # one token of one sequence without a prefix, everything in full precision: the smallest call
        {"name": "attend_one_f32", "kind": "attend", "heads": "7b", "sequences": 1, "rows": 1, "pad": 0, "type": "f32", "cache": "f32", "page": 16, "prefix": 0, "most": 577},
        # sixteen sequences behind one system prompt, as the decoder's batches are
        {"name": "attend_shared_f32_f16", "kind": "attend", "heads": "70b", "sequences": 16, "rows": 1, "pad": 0, "type": "f32", "cache": "f16", "page": 16, "prefix": 2048, "most": 1024},
        # a large batch behind a long document, long answers
        {"name": "attend_shared_bf16", "kind": "attend", "heads": "7b-gqa", "sequences": 48, "rows": 1, "pad": 0, "type": "bf16", "cache": "bf16", "page": 64, "prefix": 8192, "most": 4096},
        # drafted tokens: five rows a sequence, a prefix that ends inside a page, padding rows
        {"name": "attend_drafts_f16", "kind": "attend", "heads": "gqa-64", "sequences": 16, "rows": 5, "pad": 3, "type": "f16", "cache": "f16", "page": 32, "prefix": 1023, "most": 2048},
        # four drafts of one sequence against the logits of a small vocabulary
        {"name": "verify_one", "kind": "verify", "sequences": 1, "drafts": 4, "vocab": 32000, "target": "f32", "temperature": 0.8, "drafter": True, "ragged": False},
        # sixteen sequences of seven drafts against the logits of a large vocabulary
        {"name": "verify_batch", "kind": "verify", "sequences": 16, "drafts": 7, "vocab": 131072, "target": "f32", "temperature": 1.0, "drafter": True, "ragged": False},
        # probabilities, drafts of different number
        {"name": "verify_probabilities", "kind": "verify", "sequences": 64, "drafts": 4, "vocab": 32000, "target": "probabilities", "temperature": 1.0, "drafter": True, "ragged": True},
    ]


def _log(rng, low, high):
    """A whole number between low and high, its logarithm spread evenly."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "verify"])
    if kind == "verify":
        sequences, drafts = _log(rng, 1, 64), rng.randint(1, 8)
        vocab = _log(rng, 1000, max(1000, min(131072, 16 * 8 * 131072 // (sequences * (drafts + 1)))))
        target = rng.choice(["f32", "f32", "bf16", "f16", "probabilities"])
        return {"kind": kind, "sequences": sequences, "drafts": drafts, "vocab": vocab, "target": target,
                "temperature": 1.0 if target == "probabilities" else rng.choice([0.0, 0.6, 1.0, 1.3]), "drafter": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    heads = rng.choice(sorted(HEADS))
    h, kv, hd = HEADS[heads]
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
    how = {"rot": rng.choice([hd, hd // 2]), "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "llama3", "yarn"])}
    if kind == "rope":
        batch = _log(rng, 1, 16)
        seq = _log(rng, 1, max(1, 4096 * 72 * 128 * 2 // ((h + kv) * hd * BYTES[act] * batch)))
        return {"kind": kind, "heads": heads, "batch": batch, "seq": seq, "type": act, **how, "backward": rng.random() < 0.4}
    page = rng.choice([16, 32, 64, 128])
    prefix = 0 if rng.random() < 0.25 else _log(rng, 17, 8192)
    if kind == "append":
        sequences = _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, 8190 // sequences))
        return {"kind": kind, "heads": heads, "sequences": sequences, "rows": rows, "pad": rng.choice([0, 0, 1, 5]), "type": act, "cache": cache, "page": page, "prefix": prefix,
                "most": 2 * rows + rng.randint(1, 300), **how}
    sequences = _log(rng, 1, 48)
    rows = 1 if rng.random() < 0.6 else rng.randint(2, 8)
    room = 48 * 4096 * 8 * 128 // (sequences * rows * kv * hd)  # keys a sequence, where the plain form holds them for every row
    return {"kind": kind, "heads": heads, "sequences": sequences, "rows": rows, "pad": rng.choice([0, 0, 3]), "type": act, "cache": cache, "page": page,
            "prefix": min(prefix, 8192 * 8 * 128 // (kv * hd)), "most": _log(rng, min(16, room), min(4096, room))}


def _spread(most, count):
    """How long each of `count` sequences is: from a quarter of the longest on, evenly."""
    return [most - (3 * most * i) // (4 * max(1, count - 1)) if count > 1 else most for i in range(count)]


def _rows_of(case):
    """New rows of each sequence: the same number for steps, ragged for prompts."""
    n, rows = case["sequences"], case["rows"]
    return [rows] * n if rows <= 8 else [max(1, rows + (i % 5 - 2) * rows // 9) for i in range(n)]


def _scaled(kind):
    """Arguments of the scaling, of contexts of 8192 positions stretched to the table's."""
    return {"none": None, "linear": (4.0,), "llama3": (8.0, 1.0, 4.0, 8192), "yarn": (4.0, 8192)}[kind]


def _rope_handle(case):
    from jitnn_b200 import Rope, RopeScaling
    how = case["scaling"]
    scaling = None if how == "none" else getattr(RopeScaling, how)(*_scaled(how))
    return Rope(POSITIONS, case["rot"], base=BASE, scaling=scaling, interleaved=case["interleaved"], device=0)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}

    def normal(*shape, kind="f32", size=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * size).to(TYPES[kind])

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["kind"] == "verify":
        b, k, v = case["sequences"], case["drafts"], case["vocab"]
        logits = normal(b, k + 1, v, size=3.0)
        t = case["temperature"] or 1.0
        q = torch.softmax((logits[:, :k] + normal(b, k, v, size=0.8)) / t, -1)
        s["drafts"] = torch.multinomial(q.view(b * k, v), 1, generator=g).view(b, k).int()
        if not case["drafter"] or not case["temperature"]:  # drafts that are sure of themselves: mostly the likeliest token
            best = logits[:, :k].argmax(-1).int()
            s["drafts"] = torch.where(torch.rand(b, k, generator=g, device="cuda") < 0.8, best, s["drafts"])
        s["q"] = q if case["drafter"] and case["temperature"] else None
        s["u"] = torch.rand(b, k + 1, generator=g, device="cuda")
        s["counts"] = torch.randint(0, k + 1, (b,), generator=g, device="cuda").int() if case["ragged"] else None
        s["target"] = torch.softmax(logits, -1) if case["target"] == "probabilities" else logits.to(TYPES[case["target"]])
        s["temperature"] = None if case["target"] == "probabilities" else case["temperature"]
        return s
    h, kv, hd = HEADS[case["heads"]]
    if case["kind"] == "rope":
        b, t = case["batch"], case["seq"]
        s["q"], s["k"] = normal(b, t, h, hd, kind=case["type"]), normal(b, t, kv, hd, kind=case["type"])
        first = torch.randint(0, POSITIONS - t + 1, (b, 1), generator=g, device="cuda")
        s["positions"] = (first + torch.arange(t, device="cuda")).int()
        if own:
            s["rope"] = _rope_handle(case)
        return s
    n, page, prefix = case["sequences"], case["page"], case["prefix"]
    rows = _rows_of(case)
    order = torch.randperm(n, generator=g, device="cuda").tolist()
    lengths = [_spread(case["most"], n)[i] for i in order]
    lengths = [max(m, r) for m, r in zip(lengths, rows)]
    width, ahead = -(-max(lengths) // page), -(-prefix // page)
    pages = n * width + ahead + 3
    free = torch.randperm(pages, generator=g, device="cuda").int()
    tokens = sum(rows) + case["pad"]
    s["tables"] = free[: n * width].view(n, width).contiguous()
    s["prefix"] = free[n * width: n * width + ahead].contiguous() if prefix else None
    s["lengths"] = whole(lengths)
    s["starts"] = whole([sum(rows[:i]) for i in range(n + 1)])
    s["q"] = normal(tokens, h, hd, kind=case["type"])
    s["keys"], s["values"] = normal(pages, kv, page, hd, kind=case["cache"]), normal(pages, kv, page, hd, kind=case["cache"])
    if case["kind"] == "append":
        s["k"], s["v"] = normal(tokens, kv, hd, kind=case["type"]), normal(tokens, kv, hd, kind=case["type"])
    if own:
        from jitnn_b200 import PagedBatch, PagedCache
        s["pages"] = PagedCache(pages, page, kv, hd, dtype=TYPES[case["cache"]], device=0, k=s["keys"], v=s["values"])
        s["batch"] = PagedBatch(s["tables"], s["starts"], s["lengths"], prefix=s["prefix"], prefix_length=prefix)
        if case["kind"] == "append":
            s["rope"] = _rope_handle(case)
    return s


def _frequencies(case):
    """The angle per position of each pair, and the factor of the rotated values, in 64 bits."""
    rot, how = case["rot"], case["scaling"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = BASE ** (-2.0 * i / rot)
    if how == "linear":
        return f / _scaled(how)[0], 1.0
    if how == "llama3":
        factor, low, high, context = _scaled(how)
        blend = ((context * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)  # turns within the trained context
        return f * (blend + (1 - blend) / factor), 1.0
    if how == "yarn":
        factor, context = _scaled(how)
        pair = [rot * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
        keep = 1 - ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rotated(x, positions, case, sign=1.0):
    """x [..., heads, head size] in 32 bits, rotated at `positions` [...]."""
    f, size = _frequencies(case)
    angle = positions.double()[..., None, None] * f
    c, z = (angle.cos() * size).float(), (angle.sin() * size * sign).float()
    rot, x = case["rot"], x.float()
    first, rest = x[..., :rot], x[..., rot:]
    if case["interleaved"]:
        a, b = first[..., 0::2], first[..., 1::2]
        y = torch.stack((a * c - b * z, a * z + b * c), -1).flatten(-2)
    else:
        a, b = first[..., : rot // 2], first[..., rot // 2:]
        y = torch.cat((a * c - b * z, a * z + b * c), -1)
    return torch.cat((y, rest), -1)


def _of_rows(s):
    """For every row: its sequence, its position among the sequence's own keys, and whether it belongs to a sequence."""
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    real = seq < s["lengths"].numel()
    seq = seq.clamp(max=s["lengths"].numel() - 1)
    new = s["starts"][1:] - s["starts"][:-1]
    return seq, (s["lengths"] - new)[seq].long() + row - s["starts"][seq], real


def _plain_append(s):
    case = s["case"]
    seq, at, real = _of_rows(s)
    q, k = (_rotated(s[x], at + case["prefix"], case) for x in ("q", "k"))
    page = s["tables"][seq, at.clamp(min=0, max=s["tables"].shape[1] * case["page"] - 1) // case["page"]].long()
    page, slot = page[real], (at % case["page"])[real]
    s["keys"][page, :, slot] = k[real].to(s["keys"].dtype)
    s["values"][page, :, slot] = s["v"][real].to(s["values"].dtype)
    return {"q": (q * real[:, None, None]).to(s["q"].dtype), "k": s["keys"], "v": s["values"]}


def _plain_attend(s):
    case = s["case"]
    h, kv, hd = HEADS[case["heads"]]
    seq, at, real = _of_rows(s)
    q = s["q"].float().view(-1, kv, h // kv, hd) / math.sqrt(hd)
    held = s["tables"][seq].long()
    k, v = (s[x][held].float().permute(0, 2, 1, 3, 4).flatten(2, 3) for x in ("keys", "values"))  # [row, key/value head, key, head size]
    own_scores = torch.matmul(q, k.transpose(-1, -2))
    seen = torch.arange(k.shape[2], device="cuda") <= at[:, None]
    scores = [own_scores.masked_fill(~seen[:, None, None], -math.inf)]
    if case["prefix"]:
        ahead = s["prefix"].long()
        pk, pv = (s[x][ahead].float().permute(1, 0, 2, 3).flatten(1, 2)[:, : case["prefix"]] for x in ("keys", "values"))
        rows = q.permute(1, 0, 2, 3).flatten(1, 2)  # all rows of a key/value head
        scores.insert(0, torch.matmul(rows, pk.transpose(-1, -2)).view(kv, -1, h // kv, case["prefix"]).permute(1, 0, 2, 3))
    top = torch.cat([x.amax(-1, keepdim=True) for x in scores], -1).amax(-1, keepdim=True)
    weights = [(x - top).exp() for x in scores]
    total = sum(x.sum(-1, keepdim=True) for x in weights)
    out = torch.matmul(weights[-1], v)
    if case["prefix"]:
        w = weights[0].permute(1, 0, 2, 3).flatten(1, 2)
        out = out + torch.matmul(w, pv).view(kv, -1, h // kv, hd).permute(1, 0, 2, 3)
    out = (out / total).reshape(-1, h, hd) * real[:, None, None]
    return out.to(s["q"].dtype)


def _plain_verify(s):
    target, drafts, u = s["target"].double(), s["drafts"].long(), s["u"].double()
    b, k = drafts.shape
    v = target.shape[-1]
    counts = s["counts"].long() if s["counts"] is not None else torch.full((b,), k, device="cuda")
    index, each, place = torch.arange(v, device="cuda"), torch.arange(b, device="cuda"), torch.arange(k + 1, device="cuda")
    within = place[:k] < counts[:, None]
    if s["temperature"] == 0:
        best = torch.where(target == target.amax(-1, keepdim=True), index, v).amin(-1)
        accepted = ((drafts == best[:, :k]) & within).long().cumprod(1).sum(1)
        token = best[each, accepted]
    else:
        if s["temperature"] is not None:
            p = ((target - target.amax(-1, keepdim=True)) / s["temperature"]).exp()
            p = p / p.sum(-1, keepdim=True)
        else:
            p = target
        px = p[:, :k].gather(-1, drafts[..., None])[..., 0]
        qx = s["q"].double().gather(-1, drafts[..., None])[..., 0] if s["q"] is not None else torch.ones_like(px)
        accepted = ((u[:, :k] * qx < px) & within).long().cumprod(1).sum(1)
        last = accepted.clamp(max=k - 1)
        q = s["q"][each, last].double() if s["q"] is not None else (index == drafts[each, last][:, None]).double()
        p = p[each, accepted]
        rest = (p - q * (accepted < counts)[:, None]).clamp(min=0)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
        upto = rest.cumsum(-1)
        token = (upto <= u[:, k:] * upto[:, -1:]).sum(-1).clamp(max=v - 1)
    drafts = torch.cat((drafts, drafts[:, :1]), 1)
    tokens = torch.where(place < accepted[:, None], drafts, torch.where(place == accepted[:, None], token[:, None], -1))
    return {"accepted": accepted.int(), "tokens": tokens.int()}


def run(s):
    case = s["case"]
    if case["kind"] == "rope":
        if own:
            turn = s["rope"].backward if case["backward"] else s["rope"].rotate
            return turn((s["q"], s["k"]), s["positions"])
        sign = -1.0 if case["backward"] else 1.0
        return tuple(_rotated(x, s["positions"], case, sign).to(x.dtype) for x in (s["q"], s["k"]))
    if case["kind"] == "append":
        if own:
            q = s["pages"].append(s["q"], s["k"], s["v"], s["batch"], rope=s["rope"])
            return {"q": q, "k": s["pages"].k, "v": s["pages"].v}
        return _plain_append(s)
    if case["kind"] == "attend":
        return s["pages"].attention(s["q"], s["batch"]) if own else _plain_attend(s)
    if own:
        from jitnn_b200 import Speculative
        accepted, tokens = Speculative.verify(s["target"], s["drafts"], s["u"], draft_probs=s["q"], counts=s["counts"], temperature=s["temperature"])
        return {"accepted": accepted, "tokens": tokens}
    return _plain_verify(s)


def work(case):
    if case["kind"] == "verify":
        b, k, v = case["sequences"], case["drafts"], case["vocab"]
        row = v * BYTES.get(case["target"], 4)
        if case["target"] == "probabilities":  # the drafts' probabilities, and the row that is drawn from
            return {"bytes": b * (row + (4 * v if case["drafter"] else 0) + 24 * (k + 1)), "flops": 3.0 * b * v}
        drawn = 4 * v if case["drafter"] and case["temperature"] else 0
        return {"bytes": b * ((k + 1) * row + drawn + 24 * (k + 1)), "flops": b * ((k + 1) * 12.0 * v + 3.0 * v)}
    h, kv, hd = HEADS[case["heads"]]
    if case["kind"] == "rope":
        tokens = case["batch"] * case["seq"]
        return {"bytes": tokens * ((h + kv) * hd * 2 * BYTES[case["type"]] + 4), "flops": 3.0 * tokens * (h + kv) * case["rot"]}
    rows, tokens = _rows_of(case), sum(_rows_of(case))
    if case["kind"] == "append":
        moved = tokens * ((2 * h + 2 * kv) * hd * BYTES[case["type"]] + 2 * kv * hd * BYTES[case["cache"]])
        return {"bytes": moved + 4 * (tokens + 3 * case["sequences"]), "flops": 3.0 * tokens * (h + kv) * case["rot"]}
    lengths = [max(m, r) for m, r in zip(_spread(case["most"], case["sequences"]), rows)]
    held = (case["prefix"] + sum(lengths)) * kv * hd * 2 * BYTES[case["cache"]]
    pairs = sum(r * (case["prefix"] + m) - r * (r - 1) // 2 for m, r in zip(lengths, rows))
    return {"bytes": held + 2 * tokens * h * hd * BYTES[case["type"]], "flops": 4.0 * pairs * h * hd}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return None  # whole numbers
    h, kv, hd = HEADS[case["heads"]]

    def turned(x, positions, back=False):
        """x as complex numbers, times e^(i angle)."""
        f, size = _exact_frequencies(case)
        by = torch.polar(torch.full((1,), size, dtype=torch.float64, device="cuda"), positions.double()[..., None] * f * (-1 if back else 1))[..., None, :]
        x, rot = x.double(), case["rot"]
        pairs = x[..., :rot].unflatten(-1, (rot // 2, 2)) if case["interleaved"] else x[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, x[..., rot:]), -1)

    if case["kind"] == "rope":
        return tuple(turned(s[x], s["positions"], case["backward"]) for x in ("q", "k"))
    starts, lengths, page, prefix = s["starts"].tolist(), s["lengths"].tolist(), case["page"], case["prefix"]
    if case["kind"] == "append":
        q, keys, values = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), s["keys"].double(), s["values"].double()
        for i, total in enumerate(lengths):
            rows = slice(starts[i], starts[i + 1])
            at = torch.arange(total - starts[i + 1] + starts[i], total, device="cuda")
            q[rows] = turned(s["q"][rows], at + prefix)
            where = s["tables"][i].long()[at // page], slice(None), at % page
            keys[where] = turned(s["k"][rows], at + prefix)
            values[where] = s["v"][rows].double()
        return {"q": q, "k": keys, "v": values}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, total in enumerate(lengths):
        n = starts[i + 1] - starts[i]
        held = [s["tables"][i, : -(-total // page)]] + ([s["prefix"]] if prefix else [])
        k, v = ([s[x][p.long()].transpose(0, 1).reshape(kv, -1, hd)[:, :m] for p, m in zip(held, (total, prefix))] for x in ("keys", "values"))
        k, v = (torch.cat(x, 1).double() for x in (k, v))
        q = s["q"][starts[i]: starts[i + 1]].double().view(n, kv, h // kv, hd)
        score = torch.einsum("nkgd,kjd->nkgj", q, k) / math.sqrt(hd)
        j = torch.arange(k.shape[1], device="cuda")
        hidden = (j < total) & (j > total - n + torch.arange(n, device="cuda")[:, None])
        out[starts[i]: starts[i + 1]] = torch.einsum("nkgj,kjd->nkgd", torch.softmax(score.masked_fill(hidden[:, None, None], -math.inf), -1), v).reshape(n, h, hd)
    return out


def _exact_frequencies(case):
    """The definition, one pair after the other."""
    rot, how = case["rot"], case["scaling"]
    got, size = [], 1.0
    for i in range(rot // 2):
        f = math.exp(-2.0 * i / rot * math.log(BASE))
        if how == "linear":
            f /= _scaled(how)[0]
        elif how == "llama3":
            factor, low, high, context = _scaled(how)
            wave = 2 * math.pi / f
            if wave > context / low:
                f /= factor
            elif wave >= context / high:
                smooth = (context / wave - low) / (high - low)
                f = (1 - smooth) * f / factor + smooth * f
        elif how == "yarn":
            factor, context = _scaled(how)
            size = 1.0 + 0.1 * math.log(factor)
            first = max(0, math.floor(rot / 2 * math.log(context / (2 * math.pi * 32.0), BASE)))
            last = min(rot - 1, math.ceil(rot / 2 * math.log(context / (2 * math.pi), BASE)))
            part = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = f / factor * part + f * (1 - part)
        got.append(f)
    return torch.tensor(got, dtype=torch.float64, device="cuda"), size

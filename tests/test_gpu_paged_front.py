"""Operators of paged decoding: the native front against the general code in paged.py, and calls as a program makes them: first of all in a capture, from threads, in a row, twice at once."""
import subprocess
import sys
import threading

import pytest
import torch

import paged_oracle as oracle
from conftest import ROOT
from jitnn_b200 import PagedBatch, PagedCache, Rope, Speculative, device_status, ops

pytestmark = pytest.mark.gpu
F32, F16, BF16, I32 = torch.float32, torch.float16, torch.bfloat16, torch.int32


class Slow:
    """paged without the front."""
    def __enter__(self):
        self.front, ops._front = ops._front, None

    def __exit__(self, *a):
        ops._front = self.front


def both(call):
    assert ops._front is not None
    fast = call()
    with Slow():
        slow = call()
    fast, slow = ((x if isinstance(x, tuple) else (x,)) for x in (fast, slow))
    assert len(fast) == len(slow)
    for x, y in zip(fast, slow):
        assert type(x) is torch.Tensor and x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and x.device == y.device
        assert torch.equal(x.view(torch.uint8) if x.dtype != I32 else x, y.view(torch.uint8) if y.dtype != I32 else y)


def whole(*x):
    return torch.tensor(x, dtype=I32, device="cuda")


def made(cache=F16, act=F32, kv=2, hd=64, tokens=7):
    g = torch.Generator("cuda").manual_seed(3)
    pages = PagedCache(20, 16, kv, hd, dtype=cache, k=torch.randn(20, kv, 16, hd, generator=g, device="cuda").to(cache), v=torch.randn(20, kv, 16, hd, generator=g, device="cuda").to(cache))
    batch = PagedBatch(torch.arange(15, device="cuda", dtype=I32).flip(0).view(3, 5), whole(0, 1, 5, 6), whole(9, 70, 33), prefix=whole(17, 16), prefix_length=21)
    q, k, v = (torch.randn(tokens, h, hd, generator=g, device="cuda").to(act) for h in (4 * kv, kv, kv))
    return pages, batch, Rope(200, hd), q, k, v


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
def test_the_same_bits(act, cache):
    pages, batch, rope, q, k, v = made(cache, act)
    at = torch.arange(7, device="cuda")
    fused = torch.cat((q, k, v), 1)
    for x in (q, fused[:, :8], q.transpose(0, 1).contiguous().transpose(0, 1)):
        both(lambda: rope.rotate(x, at))
        both(lambda: rope.rotate((x, k), at.int()))
        both(lambda: rope.backward((x,), 5))
        both(lambda: rope.rotate(x.unsqueeze(0), at))
        both(lambda: pages.append(x, k, v, batch, rope=rope))
        both(lambda: pages.append(x, fused[:, 8:10], fused[:, 10:], batch))
        both(lambda: pages.attention(x, batch))
        both(lambda: pages.attention(x, batch, scale=0.3))
    both(lambda: rope.rotate(q[:0], at[:0]))
    both(lambda: pages.attention(q[:0], batch))
    assert device_status(0) == 0


@pytest.mark.parametrize("target", [F32, F16, BF16, "probabilities"])
@pytest.mark.parametrize("drafter,ragged", [(True, True), (False, False)])
def test_the_same_tokens(target, drafter, ragged):
    g = torch.Generator("cuda").manual_seed(4)
    x = torch.randn(5, 4, 999, generator=g, device="cuda") * 3
    x = x.softmax(-1) if target == "probabilities" else x.to(target)
    drafts = torch.randint(0, 999, (5, 3), generator=g, device="cuda", dtype=I32)
    u = torch.rand(5, 4, generator=g, device="cuda")
    q = torch.randn(5, 3, 999, generator=g, device="cuda").softmax(-1) if drafter else None
    counts = whole(3, 0, 2, 1, 3) if ragged else None
    for temperature in ((None,) if target == "probabilities" else (0.0, 0.7, 1)):
        both(lambda: Speculative.verify(x, drafts, u, q, counts, temperature))
    both(lambda: Speculative.verify(x[:0], drafts[:0], u[:0], None, None, None if target == "probabilities" else 1.0))


def test_what_is_not_plain_goes_on_to_the_general_code():
    pages, batch, rope, q, k, v = made()
    f = ops._front

    class Sub(torch.Tensor):
        pass

    for args in ((rope, q.cpu(), 0, 0), (rope, q.double(), 0, 0), (rope, q[0], 0, 0), (rope, q.as_subclass(Sub), 0, 0), (rope, q.transpose(1, 2), 0, 0), (rope, q, torch.zeros(7), 0),
                 (rope, (q, k.half()), 0, 0), (rope, [q, k, v], 0, 0), (rope, q), ("r", q, 0, 0)):
        assert f.rope(*args) is None
    for args in ((pages, q, k, v, "b", None), (pages, None, k, v, batch, None), (pages, q.half(), k, v, batch, None), (pages, q, k[1:], v, batch, None), (pages, q, k, v, batch, "r"), (pages, q, k)):
        assert f.append(*args) is None
    for args in ((pages, q, batch, 1), (pages, q.double(), batch, 1.0), (pages, q[:, :3], batch, 1.0), (batch, q, batch, 1.0), (pages, q[..., :32], batch, 1.0)):
        assert f.attention(*args) is None
    columns = q.transpose(1, 2).contiguous().transpose(1, 2)  # what the general code takes, it still takes
    assert torch.equal(pages.attention(columns, batch), pages.attention(q, batch)) and torch.equal(rope.rotate(columns, 3), rope.rotate(q, 3))
    with pytest.raises(ValueError, match="queries of shape"):
        pages.attention(q[..., :32], batch)
    rope.release()
    assert f.rope(rope, q, 0, 0) is None and f.append(pages, q, k, v, batch, rope) is None
    with pytest.raises(RuntimeError, match="released"):
        rope.rotate(q, 0)
    pages.release()
    assert f.attention(pages, q, batch, 1.0) is None
    with pytest.raises(RuntimeError, match="released"):
        pages.attention(q, batch)


def test_while_torch_calls_are_intercepted():
    from torch.utils._python_dispatch import TorchDispatchMode
    pages, batch, rope, q, k, v = made()
    want = pages.attention(q, batch), rope.rotate(q, 0)

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Dispatch():
        assert ops._front.attention(pages, q, batch, 1.0) is None and ops._front.rope(rope, q, 0, 0) is None
        assert torch.equal(pages.attention(q, batch), want[0]) and torch.equal(rope.rotate(q, 0), want[1])
    with torch.inference_mode():
        assert pages.attention(q, batch).is_inference() and rope.rotate(q, 0).is_inference()
    grown = torch.nn.Parameter(q)
    assert not pages.attention(grown, batch).requires_grad


def test_streams_and_threads():
    """Four threads on streams of their own, one cache: each the bits that it gets alone."""
    pages, batch, rope, q, k, v = made(tokens=7)
    qs = [q * (i + 1) for i in range(4)]
    x = torch.randn(4, 3, 5000, device="cuda")
    drafts, u = torch.randint(0, 5000, (4, 2), device="cuda", dtype=I32), torch.rand(4, 3, device="cuda")
    one = lambda i: (pages.attention(qs[i], batch), rope.rotate(qs[i], i), *Speculative.verify(x, drafts, u, temperature=0.5 + i))
    want = [one(i) for i in range(4)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(100):
                got = one(i)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert bad == [] and device_status(0) == 0


def test_a_generation_step_in_a_graph_beside_another():
    """Append, attention and verification captured together, twice; both graphs replayed on two streams at once, over lengths that change between the replays."""
    steps = []
    for seed in (1, 2):
        pages, batch, rope, q, k, v = made()
        x = torch.randn(3, 5, 700, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
        drafts, u = torch.randint(0, 700, (3, 4), device="cuda", dtype=I32), torch.rand(3, 5, device="cuda")

        def step(pages=pages, batch=batch, rope=rope, q=q, k=k, v=v, x=x, drafts=drafts, u=u):
            turned = pages.append(q, k, v, batch, rope=rope)
            return pages.attention(turned, batch), *Speculative.verify(x, drafts, u, temperature=0.9)

        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        steps.append((g, out, step, batch, torch.cuda.Stream()))
    for lengths in ((9, 70, 33), (1, 4, 1), (80, 5, 80), (9, 70, 33)):
        for _, _, _, batch, _ in steps:
            batch.lengths.copy_(whole(*lengths))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, _, _, _, s in steps:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        got = [[y.clone() for y in out] for _, out, _, _, _ in steps]
        for (_, _, step, _, _), seen in zip(steps, got):
            for a, b in zip(step(), seen):
                assert torch.equal(a, b)
    assert device_status(0) == 0


@pytest.mark.parametrize("captured", [False, True])
def test_kernels_in_front_and_on_other_streams(captured):
    """Calls behind kernels that make their inputs, row after row of them, and behind two streams at once; what comes behind them sees their results."""
    pages, batch, rope, q, k, v = made(act=F16, cache=F16)
    fixed = [q * (i + 1) for i in range(6)]
    want = [pages.attention(rope.rotate(x, 3), batch) for x in fixed]
    u, drafts = torch.rand(3, 2, device="cuda"), torch.zeros(3, 1, dtype=I32, device="cuda")
    logits = torch.randn(3, 2, 40000, device="cuda")
    tokens = Speculative.verify(logits * 2, drafts, u, temperature=1.0)[1]
    side, buffer, lengths = torch.cuda.Stream(), torch.empty_like(q), batch.lengths.clone()
    torch.cuda.synchronize()

    def run():
        got, here = [], torch.cuda.current_stream()
        for x in fixed:
            side.wait_stream(here)
            with torch.cuda.stream(side):
                batch.lengths.zero_()
                batch.lengths.add_(lengths)
            buffer.fill_(7.0)
            buffer.copy_(x)
            turned = rope.rotate(buffer, 3)
            here.wait_stream(side)
            got.append(pages.attention(turned, batch) * 1)
            batch.lengths.zero_()
            batch.lengths.add_(lengths)
            got.append(pages.attention(rope.rotate(buffer, 3), batch))
            got.append(Speculative.verify(logits + logits, drafts, u, temperature=1.0)[1] + 0)
        return got

    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run()
        for _ in range(20):
            g.replay()
    else:
        for _ in range(20):
            got = run()
    torch.cuda.synchronize()
    for i in range(6):
        assert torch.equal(got[3 * i], want[i]) and torch.equal(got[3 * i + 1], want[i]) and torch.equal(got[3 * i + 2], tokens)


def test_what_is_read_later_is_not_copied():
    """A batch's numbers are read when the kernels run: changed in place they count, and tensors that would have to be copied are refused."""
    pages, batch, rope, q, k, v = made()
    before = pages.attention(q, batch)
    batch.lengths.copy_(whole(9, 70, 1))
    after, again = pages.attention(q, batch), pages.attention(q, PagedBatch(batch.tables, batch.starts, whole(9, 70, 1), prefix=batch.prefix, prefix_length=21))
    assert torch.equal(after, again) and not torch.equal(after, before)
    numbers = torch.zeros(4, 2, dtype=I32, device="cuda")
    for change in ({"starts": numbers[:, 0]}, {"lengths": numbers[:3, 1]}, {"tables": batch.tables.t().contiguous().t()}, {"prefix": numbers[:2, 0], "prefix_length": 21}):
        args = {"tables": batch.tables, "starts": batch.starts, "lengths": batch.lengths, **change}
        with pytest.raises(ValueError, match="strides"):
            PagedBatch(**args)


def test_scales_that_are_no_numbers_are_refused():
    pages, batch, rope, q, k, v = made()
    for scale in (float("nan"), float("inf"), 1e39, 3e38):
        with pytest.raises(ValueError, match="scale"):
            pages.attention(q, batch, scale=scale)
        with Slow(), pytest.raises(ValueError, match="scale"):
            pages.attention(q, batch, scale=scale)


def test_two_rows_for_one_place():
    """Two sequences on the same pages: where both write, either's key may stand, whole."""
    pages, _, _, q, k, v = made()
    tables = whole(3, 4).view(1, 2).expand(2, 2)
    batch = PagedBatch(tables, whole(0, 1, 2), whole(5, 5))
    for _ in range(5):
        pages.append(None, k[:2], v[:2], batch)
        for stored, new in ((pages.k, k), (pages.v, v)):
            got = stored[3, :, 4]
            assert all(any(torch.equal(got[h], new[r, h].half()) for r in range(2)) for h in range(2))
    assert device_status(0) == 0


FIRST = """
import sys; sys.path[:0] = [%r, %r]
import torch
from jitnn_b200 import Speculative
x, drafts, u = torch.randn(2, 3, 500, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.rand(2, 3, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = Speculative.verify(x, drafts, u, temperature=1.0)
g.replay()
want = Speculative.verify(x, drafts, u, temperature=1.0)
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("the same")
""" % (ROOT, ROOT + "/tests")


FIRST_STEP = """
import sys; sys.path[:0] = [%r, %r]
import torch
from jitnn_b200 import PagedBatch, PagedCache, Rope
whole = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
for hd, tokens in ((64, 1), (128, 40)):
    k, v = (torch.randn(20, 1, 16, hd, device="cuda").half() for _ in range(2))
    pages, rope = PagedCache(20, 16, 1, hd, dtype="F16", k=k, v=v), Rope(400, hd)
    batch = PagedBatch(torch.arange(10, device="cuda", dtype=torch.int32).view(1, 10), whole(0, tokens), whole(100), prefix=torch.arange(10, 20, device="cuda", dtype=torch.int32), prefix_length=150)
    q, n = torch.randn(tokens, 4, hd, device="cuda").half(), torch.randn(tokens, 1, hd, device="cuda").half()
    step = lambda: pages.attention(pages.append(rope.rotate(q, 0), n, n, batch, rope=rope), batch)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    assert torch.equal(got, step()) and torch.isfinite(got).all()
print("the same")
""" % (ROOT, ROOT + "/tests")


@pytest.mark.parametrize("program", [FIRST, FIRST_STEP], ids=["verification", "step"])
def test_the_first_call_of_a_process_in_a_capture(program):
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]

"""Operators of paged decoding on torch CUDA tensors: rotary positions, a paged cache of keys and values with the attention that reads it, and the verification of
drafted tokens (the jq_rope_*, jq_pages_* and jq_verify_* entry points of the C ABI, whose header says what each computes).

``Rope`` and ``RopeScaling`` follow ops/Rope.java:84-149 of the reference (``F.ropeHeads`` with its ``RopeScaling``); the reference has neither a cache nor a generation
loop, the rest has no counterpart there. All calls are enqueued on torch's current stream of the tensors' device and may be captured into a CUDA graph: what they need
beside their arguments is allocated by torch for that call.
"""
import ctypes
import math

from . import _lib, ops
from ._lib import check
from .ops import _raw_stream, _t

# The plain calls, with outputs of their own, are methods of the native front (csrc/front.cpp) where there is one; it hands back None for everything else, which goes on here.

_ELEM = {"F32": 0, "F16": 1, "BF16": 2}


def _elem(dtype):
    """(code, torch type) of a torch floating type or of "F32", "F16", "BF16"."""
    torch = _t()
    types = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
    for name, t in types.items():
        if dtype is t or dtype == name:
            return _ELEM[name], t
    raise ValueError("needs an FP32, FP16 or BF16 tensor, got %s" % (dtype,))


def _cuda(x, what, device, dims):
    """Checks that x is a CUDA tensor of `dims` axes on `device` with its last axis in one piece; returns it, or a contiguous copy."""
    torch = _t()
    if not isinstance(x, torch.Tensor):
        raise ValueError("%s: a torch CUDA tensor is needed, got %s" % (what, type(x).__name__))
    if x.dim() not in dims:
        raise ValueError("%s of shape %s" % (what, list(x.shape)))
    if x.get_device() != device:
        raise ValueError("%s on %s, needed on cuda:%d" % (what, x.device, device))
    return x if x.stride(-1) == 1 else x.contiguous()


def _whole(x, what, device, shape, copy=True):
    """An int32 CUDA tensor of that shape on `device`, contiguous, of which without `copy` nothing else may be made: it is read later."""
    torch = _t()
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32:
        raise ValueError("%s: an int32 CUDA tensor is needed, got %s" % (what, x.dtype if isinstance(x, torch.Tensor) else type(x).__name__))
    if tuple(x.shape) != tuple(shape):
        raise ValueError("%s of shape %s, needed %s" % (what, list(x.shape), list(shape)))
    if x.get_device() != device:
        raise ValueError("%s on %s, needed on cuda:%d" % (what, x.device, device))
    if not copy and not x.is_contiguous():
        raise ValueError("%s of strides %s, needed contiguous" % (what, list(x.stride())))
    return x.contiguous()


def _span(x):
    """The bytes from x's first element to behind its last."""
    return x.data_ptr(), x.data_ptr() + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size() if x.numel() else x.data_ptr()


def _overlap(x, y):
    a, b = _span(x), _span(y)
    return a[0] < b[1] and b[0] < a[1]


def _output(out, x, what):
    """`out`, checked against x, which it may be, but not overlap otherwise; or a new tensor."""
    if out is None:
        return x.new_empty(x.shape)
    if out.dtype is not x.dtype or out.shape != x.shape or out.get_device() != x.get_device():
        raise ValueError("%s: output %s %s for %s %s" % (what, out.dtype, list(out.shape), x.dtype, list(x.shape)))
    if out.numel() and out.stride(-1) != 1 or any(s == 0 and n > 1 for n, s in zip(out.shape, out.stride())):
        raise ValueError("%s: output of strides %s" % (what, list(out.stride())))
    if not (out.data_ptr() == x.data_ptr() and out.stride() == x.stride()):
        if _overlap(out, x):
            raise ValueError("%s: the output overlaps the input and is not the input" % what)
    return out


class RopeScaling:
    """How the frequencies of a rotation are rescaled for contexts longer than the trained one."""

    def __init__(self, kind, *params):
        self.kind, self.params = kind, tuple(float(p) for p in params)

    @staticmethod
    def linear(factor):
        """Every position divided by `factor`."""
        return RopeScaling(1, factor)

    @staticmethod
    def llama3(factor, low, high, context):
        """Pairs with fewer than `low` turns in `context` positions slowed down by `factor`, with more than `high` as they were, linear between."""
        return RopeScaling(2, factor, low, high, context)

    @staticmethod
    def yarn(factor, context, fast=32.0, slow=1.0, magnitude=0.0):
        """The same between the pairs that make `fast` and `slow` turns, and rotated values times `magnitude` (0: 0.1 ln(factor) + 1)."""
        return RopeScaling(3, factor, context, fast, slow, magnitude)

    @staticmethod
    def frequencies(dim, base=10000.0, scaling=None):
        """(angles per position of the dim / 2 pairs, magnitude) as Python floats."""
        freqs, magnitude = (ctypes.c_double * max(1, dim // 2))(), ctypes.c_double()
        kind, params = (0, ()) if scaling is None else (scaling.kind, scaling.params)
        check(_lib.load().jq_rope_frequencies(dim, base, kind, (ctypes.c_double * 5)(*params), freqs, ctypes.byref(magnitude)))
        return list(freqs[: dim // 2]), magnitude.value


class Rope:
    """A table of rotations for positions 0 .. positions - 1 on one GPU; pairs are (x[i], x[i + dim / 2]), or next to each other where ``interleaved``.

    Only the first ``dim`` elements of a head are rotated, the others are copied."""

    def __init__(self, positions, dim, base=10000.0, scaling=None, interleaved=False, device=0):
        self._h = None
        freqs, magnitude = RopeScaling.frequencies(dim, base, scaling)
        h = ctypes.c_void_p()
        check(_lib.load().jq_rope_create(device, positions, dim, (ctypes.c_double * len(freqs))(*freqs), magnitude, int(interleaved), ctypes.byref(h)))
        self._h, self.positions, self.dim, self.device = h, positions, dim, device
        self._addr = h.value

    def _handle(self):
        if self._h is None:
            raise RuntimeError("the rotation was released")
        return self._h

    def rotate(self, x, positions, out=None):
        """x [tokens, heads, head size] or [batch, tokens, heads, head size], or a pair of such (queries, keys), rotated. ``positions``: an int32 or int64 CUDA tensor
        [tokens] or [batch, tokens], or the int position of the first token. ``out`` may be x."""
        if ops._front is not None and out is None:
            y = ops._front.rope(self, x, positions, 0)
            if y is not None:
                return y
        return self._turn(x, positions, out, 0, "rotation")

    def backward(self, g, positions, out=None):
        """The gradient of x from the gradient of ``rotate(x, positions)``."""
        if ops._front is not None and out is None:
            y = ops._front.rope(self, g, positions, 1)
            if y is not None:
                return y
        return self._turn(g, positions, out, 1, "rotation backward")

    def _turn(self, x, positions, out, inverse, what):
        torch = _t()
        h = self._handle()
        pair = isinstance(x, (tuple, list))
        xs = tuple(x) if pair else (x,)
        outs = (tuple(out) if pair else (out,)) if out is not None else (None,) * len(xs)
        if len(xs) not in (1, 2) or len(outs) != len(xs):
            raise ValueError("%s: %d tensors, %d outputs (one tensor, or queries and keys)" % (what, len(xs), len(outs)))
        xs = tuple(_cuda(t, what + ": input", self.device, (3, 4)) for t in xs)
        code, _ = _elem(xs[0].dtype)
        lead, hd = tuple(xs[0].shape[:-2]), xs[0].shape[-1]
        for t in xs[1:]:
            if tuple(t.shape[:-2]) != lead or t.shape[-1] != hd or t.dtype is not xs[0].dtype:
                raise ValueError("%s: %s %s beside %s %s" % (what, t.dtype, list(t.shape), xs[0].dtype, list(xs[0].shape)))
        ys = tuple(_output(o, t, what) for o, t in zip(outs, xs))
        if len(xs) == 2 and all(t.numel() for t in xs) and (ys[0].data_ptr() in (ys[1].data_ptr(), xs[1].data_ptr()) or ys[1].data_ptr() == xs[0].data_ptr()):
            raise ValueError("%s: one tensor is the other's output" % what)
        batch, seq = (1,) + lead if len(lead) == 1 else lead
        at, size, pb, pt, offset = None, 0, 0, 0, 0
        if isinstance(positions, torch.Tensor):
            if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in (lead, lead[-1:]):
                raise ValueError("%s: positions %s %s for tokens %s" % (what, positions.dtype, list(positions.shape), list(lead)))
            if positions.get_device() != self.device:
                raise ValueError("%s: positions on %s, needed on cuda:%d" % (what, positions.device, self.device))
            at, size = positions.data_ptr(), positions.element_size()
            pb, pt = (positions.stride(0) if positions.dim() == 2 else 0), positions.stride(-1)
        else:
            offset = int(positions)
        L = _lib.load()
        turned = [p for p in zip(xs, ys) if p[0].numel()]  # (queries without keys, or keys without queries, are rotated alone)
        if turned:
            n, vps = len(turned), ctypes.c_void_p * len(turned)
            strides = (ctypes.c_int64 * (6 * n))()
            for i, t in enumerate(v for p in turned for v in p):
                strides[3 * i: 3 * i + 3] = ((0,) if len(lead) == 1 else ()) + tuple(t.stride()[:-1])
            check(L.jq_rope_apply(h, code, n, vps(*(x.data_ptr() for x, _ in turned)), vps(*(y.data_ptr() for _, y in turned)), (ctypes.c_int * n)(*(x.shape[-2] for x, _ in turned)),
                                  hd, strides, batch, seq, at, size, pb, pt, offset, inverse, _raw_stream(torch, self.device)))
        return ys if pair else ys[0]

    def release(self):
        if self._h is not None:
            h, self._h, self._addr = self._h, None, 0
            check(_lib.load().jq_rope_free(h))

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


class PagedBatch:
    """Which rows of a call belong to which sequence and where their keys lie (int32 CUDA tensors, read when the kernels run; checked here, once).

    Rows ``starts[s] .. starts[s + 1] - 1`` are the newest of sequence s, which has ``lengths[s]`` keys of its own once they are appended, key i on page
    ``tables[s, i // page_size]``. In front of them all sequences see the ``prefix_length`` keys on the pages ``prefix``. Nothing is copied: what is changed in the tensors afterwards
    counts for the calls behind."""

    def __init__(self, tables, starts, lengths, prefix=None, prefix_length=0):
        torch = _t()
        if not isinstance(tables, torch.Tensor) or tables.dim() != 2 or tables.dtype is not torch.int32 or not tables.is_cuda or 0 in tables.shape:
            raise ValueError("tables of pages: an int32 CUDA tensor [sequences, pages] is needed")
        self.device = tables.get_device()
        if tables.stride(1) != 1 and tables.shape[1] != 1:
            raise ValueError("tables of pages of strides %s (a sequence's page numbers are to be next to each other)" % list(tables.stride()))
        self.tables = tables
        sequences = tables.shape[0]
        self.starts = _whole(starts, "starts", self.device, (sequences + 1,), copy=False)
        self.lengths = _whole(lengths, "lengths", self.device, (sequences,), copy=False)
        self.prefix, self.prefix_length = None, int(prefix_length)
        if prefix is not None:
            if not isinstance(prefix, torch.Tensor) or prefix.dim() != 1:
                raise ValueError("prefix: an int32 CUDA tensor [pages] is needed")
            self.prefix = _whole(prefix, "prefix", self.device, prefix.shape, copy=False)
        if self.prefix_length < 0 or (self.prefix_length > 0 and self.prefix is None):
            raise ValueError("a prefix of %d keys on %s" % (self.prefix_length, "no pages" if self.prefix is None else "%d pages" % self.prefix.numel()))
        self._rows = (self.tables.data_ptr(), self.tables.stride(0), self.tables.shape[1], self.starts.data_ptr(), self.lengths.data_ptr(), sequences)
        self._ahead = (self.prefix.data_ptr() if self.prefix is not None else None, self.prefix.numel() if self.prefix is not None else 0, self.prefix_length)


class PagedCache:
    """Keys and values of many sequences on pages of ``page_size`` (a power of two from 16 to 1024) keys: ``k`` and ``v`` [pages, kv_heads, page_size, head_dim] of one
    type, FP32, FP16 or BF16, made here or given. Rows of the calls are FP32 or of that type."""

    def __init__(self, pages, page_size, kv_heads, head_dim, dtype="F32", device=0, k=None, v=None):
        torch = _t()
        self._h = None
        code, t = _elem(dtype)
        shape = (pages, kv_heads, page_size, head_dim)
        if (k is None) != (v is None):
            raise ValueError("a paged cache is given both keys and values, or neither")
        if min(shape) < 1:
            raise ValueError("a paged cache of %s" % list(shape))
        if k is None:
            k, v = (torch.empty(shape, dtype=t, device="cuda:%d" % device) for _ in range(2))
        for x, what in ((k, "keys"), (v, "values")):
            if not isinstance(x, torch.Tensor) or x.dtype is not t or tuple(x.shape) != shape or not x.is_contiguous() or x.get_device() != device:
                raise ValueError("%s of a paged cache: a contiguous %s CUDA tensor %s on cuda:%d is needed" % (what, t, list(shape), device))
        h = ctypes.c_void_p()
        check(_lib.load().jq_pages_create(device, code, pages, page_size, kv_heads, head_dim, k.data_ptr(), v.data_ptr(), ctypes.byref(h)))
        self._h, self.k, self.v, self.device, self.dtype = h, k, v, device, t
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self._addr, self._code, self._scale = h.value, code, 1.0 / math.sqrt(head_dim)

    def _handle(self):
        if self._h is None:
            raise RuntimeError("the paged cache was released")
        return self._h

    def _rows_of(self, x, heads, what):
        x = _cuda(x, what, self.device, (3,))
        if x.shape[-1] != self.head_dim or (heads is not None and x.shape[1] != heads):
            raise ValueError("%s of shape %s for pages of %d heads of %d" % (what, list(x.shape), self.kv_heads, self.head_dim))
        return x, _elem(x.dtype)[0]

    def _on_pages(self, batch):
        if not isinstance(batch, PagedBatch) or batch.device != self.device:
            raise ValueError("a PagedBatch on cuda:%d is needed, got %s" % (self.device, "one on cuda:%d" % batch.device if isinstance(batch, PagedBatch) else type(batch).__name__))

    def append(self, q, k, v, batch, rope=None, out=None):
        """Stores the rows k and v [tokens, kv_heads, head_dim] on their sequences' pages, k rotated by ``rope`` at each row's position, and returns q [tokens, heads,
        head_dim] rotated likewise (``out``, which may be q; None where q is None). Rows of no sequence become zero in a new tensor, and stay as they are in ``out``."""
        if ops._front is not None and out is None:
            y = ops._front.append(self, q, k, v, batch, rope)
            if y is not None:
                return y
        torch = _t()
        h = self._handle()
        self._on_pages(batch)
        k, code = self._rows_of(k, self.kv_heads, "append: keys")
        v, vcode = self._rows_of(v, self.kv_heads, "append: values")
        if vcode != code or v.shape[0] != k.shape[0]:
            raise ValueError("append: keys %s %s and values %s %s" % (k.dtype, list(k.shape), v.dtype, list(v.shape)))
        if rope is not None and (not isinstance(rope, Rope) or rope.device != self.device):
            raise ValueError("append: a Rope on cuda:%d is needed" % self.device)
        if q is None:
            heads, qp, yp, y = 0, None, None, None
            strides = (ctypes.c_int64 * 8)(0, 0, k.stride(0), k.stride(1), v.stride(0), v.stride(1), 0, 0)
        else:
            q, qcode = self._rows_of(q, None, "append: queries")
            if qcode != code or q.shape[0] != k.shape[0]:
                raise ValueError("append: queries %s %s and keys %s %s" % (q.dtype, list(q.shape), k.dtype, list(k.shape)))
            y = _output(out, q, "append")
            if y.data_ptr() != q.data_ptr() and any(_overlap(y, x) for x in (k, v)):
                raise ValueError("append: the output overlaps the keys or the values")
            heads, qp, yp = q.shape[1], q.data_ptr(), y.data_ptr()
            strides = (ctypes.c_int64 * 8)(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), y.stride(0), y.stride(1))
        if k.shape[0]:
            check(_lib.load().jq_pages_append(h, None if rope is None else rope._handle(), code, heads, qp, k.data_ptr(), v.data_ptr(), yp, strides, k.shape[0], *batch._rows,
                                              batch.prefix_length, int(out is None), _raw_stream(torch, self.device)))
        return y

    def attention(self, q, batch, scale=None, out=None):
        """softmax(scale q . k) v [tokens, heads, head_dim] of each row over the prefix and its sequence's keys up to its own; ``scale`` is 1 / sqrt(head_dim) where it
        is None. Neighbouring heads share a key/value head. A row that sees no key, or only keys with scores of negative infinity, gives zeros; rows of no sequence become zero in a new tensor, and stay as they are in ``out``."""
        scale = self._scale if scale is None else float(scale)
        if ops._front is not None and out is None:
            y = ops._front.attention(self, q, batch, scale)
            if y is not None:
                return y
        torch = _t()
        h = self._handle()
        self._on_pages(batch)
        q, code = self._rows_of(q, None, "attention: queries")
        if q.shape[1] < 1 or q.shape[1] % self.kv_heads != 0:
            raise ValueError("attention: %d query heads on %d key/value heads" % (q.shape[1], self.kv_heads))
        y = _output(out, q, "attention")
        if out is not None and q.numel() and y.data_ptr() == q.data_ptr():
            raise ValueError("attention: the output overlaps the queries")
        if q.shape[0]:
            L = _lib.load()
            need = ctypes.c_int64()
            check(L.jq_pages_attention_bytes(h, code, q.shape[1], q.shape[0], batch._rows[5], batch.prefix_length, ctypes.byref(need)))
            space = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
            strides = (ctypes.c_int64 * 4)(q.stride(0), q.stride(1), y.stride(0), y.stride(1))
            check(L.jq_pages_attention(h, code, q.shape[1], q.data_ptr(), y.data_ptr(), strides, q.shape[0], *batch._rows, *batch._ahead,
                                       scale, int(out is None), None if space is None else space.data_ptr(), need.value,
                                       _raw_stream(torch, self.device)))
        return y

    def release(self):
        if self._h is not None:
            h, self._h, self._addr = self._h, None, 0
            check(_lib.load().jq_pages_free(h))

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


class Speculative:
    """Drafted tokens against the model they were drafted for."""

    @staticmethod
    def verify(target, drafts, uniforms=None, draft_probs=None, counts=None, temperature=None):
        """(accepted [sequences], tokens [sequences, drafts + 1]), int32. ``target`` [sequences, drafts + 1, vocab]: the target's probabilities behind each draft or, with a
        ``temperature``, its logits (FP32, FP16 or BF16); ``drafts`` int32 [sequences, drafts], of which the first ``counts[s]`` are there; ``draft_probs`` FP32
        [sequences, drafts, vocab] the drafter's probabilities (None: all on the draft); ``uniforms`` FP32 [sequences, drafts + 1] in [0, 1).

        Draft i is kept while uniforms[i] q_i(x_i) < p_i(x_i), then one token is drawn at uniforms[drafts], from max(p - q, 0) behind the first refused draft and from p
        behind the last. ``tokens``: the drafts kept, that token, -1 in the rest. Temperature 0 takes the likeliest token instead and needs no uniforms. All in double."""
        temperature = None if temperature is None else float(temperature)
        if ops._front is not None:
            y = ops._front.verify(target, drafts, uniforms, draft_probs, counts, temperature)
            if y is not None:
                return y
        torch = _t()
        if not isinstance(target, torch.Tensor) or target.dim() != 3 or not target.is_cuda:
            raise ValueError("verify: a CUDA tensor [sequences, drafts + 1, vocab] of logits or probabilities is needed")
        code, _ = _elem(target.dtype)
        device = target.get_device()
        n, rows, vocab = target.shape
        if rows < 1 or vocab < 1:
            raise ValueError("verify: target of shape %s" % list(target.shape))
        target = target if target.stride(2) == 1 else target.contiguous()
        drafts = _whole(drafts, "verify: drafts", device, (n, rows - 1))
        if counts is not None:
            counts = _whole(counts, "verify: counts", device, (n,))
        logits = temperature is not None
        for x, what, shape in ((uniforms, "uniforms", (n, rows)), (draft_probs, "draft_probs", (n, rows - 1, vocab))):
            if x is None:
                continue
            if not isinstance(x, torch.Tensor) or x.dtype is not torch.float32 or tuple(x.shape) != shape or x.get_device() != device:
                raise ValueError("verify: %s: an FP32 CUDA tensor %s on cuda:%d is needed" % (what, list(shape), device))
        if uniforms is None:
            if not logits or temperature != 0:
                raise ValueError("verify: uniforms are needed unless the temperature is 0")
        else:
            uniforms = uniforms.contiguous()
        qb = qr = 0
        if draft_probs is not None:
            draft_probs = draft_probs if draft_probs.stride(2) == 1 else draft_probs.contiguous()
            qb, qr = draft_probs.stride(0), draft_probs.stride(1)
        accepted, tokens = target.new_empty((n,), dtype=torch.int32), target.new_empty((n, rows), dtype=torch.int32)
        L = _lib.load()
        need = ctypes.c_int64()
        check(L.jq_verify_bytes(n, rows - 1, vocab, int(logits), ctypes.byref(need)))
        space = torch.empty(need.value, dtype=torch.uint8, device=target.device) if need.value else None
        check(L.jq_verify_drafts(device, code, target.data_ptr(), target.stride(0), target.stride(1), drafts.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(),
                                 qb, qr, None if uniforms is None else uniforms.data_ptr(), None if counts is None else counts.data_ptr(), n, rows - 1, vocab, int(logits),
                                 temperature if logits else 0.0, accepted.data_ptr(), tokens.data_ptr(), None if space is None else space.data_ptr(), need.value,
                                 _raw_stream(torch, device)))
        return accepted, tokens

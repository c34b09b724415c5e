"""Operators of paged decoding without a GPU: the frequencies against their definitions, and calls that are refused before any device work."""
import ctypes
import math

import pytest
import torch

import paged_oracle as oracle
from jitnn_b200 import PagedBatch, PagedCache, Rope, RopeScaling, Speculative, _lib, paged
from jitnn_b200.build import build

F32, F16, I32 = torch.float32, torch.float16, torch.int32


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


@pytest.mark.parametrize("dim", [2, 6, 64, 128, 512])
@pytest.mark.parametrize("base", [1.5, 10000.0, 5e5])
@pytest.mark.parametrize("scaling,wanted", [(None, None), (RopeScaling.linear(1), ("linear", 1.0)), (RopeScaling.linear(3.5), ("linear", 3.5)),
                                            (RopeScaling.llama3(8, 1, 4, 8192), ("llama3", 8.0, 1.0, 4.0, 8192.0)), (RopeScaling.llama3(32, 0.5, 16, 64), ("llama3", 32.0, 0.5, 16.0, 64.0)),
                                            (RopeScaling.yarn(4, 4096), ("yarn", 4.0, 4096.0, 32.0, 1.0)), (RopeScaling.yarn(40, 16, 2, 0.25), ("yarn", 40.0, 16.0, 2.0, 0.25))])
def test_frequencies(lib, dim, base, scaling, wanted):
    freqs, magnitude = RopeScaling.frequencies(dim, base, scaling)
    want, want_magnitude = oracle.frequencies(dim, base, wanted)
    # a power (exponent up to 1 times ln base: 14 half steps), and in a mixture two roundings of a difference of up to 2^7 turns over low .. high
    assert freqs == pytest.approx(want, rel=1e-13, abs=0) and magnitude == pytest.approx(want_magnitude, rel=1e-15)


def test_a_magnitude_of_ones_own(lib):
    assert RopeScaling.frequencies(64, 1e4, RopeScaling.yarn(4, 4096, magnitude=0.75))[1] == 0.75


@pytest.mark.parametrize("dim,base,scaling,message", [
    (63, 1e4, None, "even"), (0, 1e4, None, "even"), (64, 1.0, None, "above 1"), (64, math.nan, None, "above 1"), (64, math.inf, None, "above 1"),
    (64, 1e4, RopeScaling.linear(0.5), "factor"), (64, 1e4, RopeScaling.linear(math.nan), "factor"), (64, 1e4, RopeScaling.llama3(8, 4, 1, 8192), "low"),
    (64, 1e4, RopeScaling.llama3(8, 1, 4, 0), "context"), (64, 1e4, RopeScaling.yarn(4, -1), "context"), (64, 1e4, RopeScaling.yarn(4, 64, 1, 1), "fast"),
    (64, 1e4, RopeScaling.yarn(4, 64, magnitude=-1), "magnitude"), (64, 1e4, RopeScaling(9, 1), "scaling 9")])
def test_frequencies_refused(lib, dim, base, scaling, message):
    with pytest.raises(ValueError, match=message):
        RopeScaling.frequencies(dim, base, scaling)


def refused(lib, rc, message):
    assert rc == _lib.JQ_ERR_INVALID and message in _lib.last_error(), (rc, _lib.last_error())


def test_handles_refused(lib):
    out, f = ctypes.c_void_p(), (ctypes.c_double * 256)()
    for positions, dim, magnitude in ((0, 64, 1.0), (2 ** 24 + 1, 64, 1.0), (16, 63, 1.0), (16, 0, 1.0), (16, 514, 1.0), (16, 64, math.nan)):
        refused(lib, lib.jq_rope_create(0, positions, dim, f, magnitude, 0, ctypes.byref(out)), "jq_rope_create")
    refused(lib, lib.jq_rope_create(0, 16, 64, None, 1.0, 0, ctypes.byref(out)), "jq_rope_create")
    refused(lib, lib.jq_rope_create(0, 16, 64, f, 1.0, 0, None), "null result")
    for elem, pages, size, heads, hd, k in ((3, 1, 16, 1, 64, 256), (-1, 1, 16, 1, 64, 256), (0, 0, 16, 1, 64, 256), (0, 2 ** 31, 16, 1, 64, 256), (0, 2 ** 30, 16, 2, 64, 256), (0, 1, 15, 1, 64, 256),
                                            (0, 1, 8, 1, 64, 256), (0, 1, 48, 1, 64, 256), (0, 1, 2048, 1, 64, 256), (0, 1, 16, 0, 64, 256), (0, 1, 16, 1025, 64, 256), (0, 1, 16, 1, 65, 256),
                                            (0, 1, 16, 1, 0, 256), (0, 1, 16, 1, 258, 256), (0, 1, 16, 1, 64, 0), (0, 1, 16, 1, 64, 264)):
        refused(lib, lib.jq_pages_create(0, elem, pages, size, heads, hd, k, 256, ctypes.byref(out)), "jq_pages_create")
    refused(lib, lib.jq_pages_create(0, 0, 1, 16, 1, 64, 256, 256, None), "null result")
    assert lib.jq_rope_free(None) == 0 and lib.jq_pages_free(None) == 0
    n = ctypes.c_int64()
    refused(lib, lib.jq_pages_attention_bytes(None, 0, 1, 1, 1, 0, ctypes.byref(n)), "not a live handle")
    dead = ctypes.create_string_buffer(4096)  # something that is no handle
    refused(lib, lib.jq_pages_free(ctypes.addressof(dead)), "not a live handle")
    refused(lib, lib.jq_rope_free(ctypes.addressof(dead)), "not a live")


@pytest.mark.parametrize("sequences,drafts,vocab", [(-1, 1, 10), (1, -1, 10), (1, 1, 0), (1, 1, 2 ** 30 + 1), (1, 4096, 10), (65536, 0, 10), (32768, 1, 10)])
def test_verification_sizes_refused(lib, sequences, drafts, vocab):
    n = ctypes.c_int64()
    refused(lib, lib.jq_verify_bytes(sequences, drafts, vocab, 1, ctypes.byref(n)), "jq_verify_drafts")
    refused(lib, lib.jq_verify_bytes(1, 1, 10, 1, None), "jq_verify_drafts")


def test_verification_workspaces(lib):
    n = ctypes.c_int64()
    for sequences, drafts, vocab in ((0, 3, 100), (1, 0, 1), (1, 4, 32000), (16, 7, 131072), (65535, 0, 7), (1, 4095, 1000), (1, 0, 2 ** 30)):
        assert lib.jq_verify_bytes(sequences, drafts, vocab, 0, ctypes.byref(n)) == 0 and n.value == 0
        assert lib.jq_verify_bytes(sequences, drafts, vocab, 1, ctypes.byref(n)) == 0
        assert 16 * sequences * (drafts + 1) <= n.value <= 16 * (sequences * (drafts + 1) * 3 + 8 * 148 * 9)  # a record for each chunk of each row


def test_verification_refused(lib):
    def call(elem=0, target=256, drafts=256, uniforms=256, logits=1, temperature=1.0, accepted=256, space=256, size=1 << 20):
        return lib.jq_verify_drafts(0, elem, target, 40, 10, drafts, None, 0, 0, uniforms, None, 2, 3, 10, logits, temperature, accepted, 256, space, size, None)

    for change, message in (({"elem": 3}, "element type"), ({"target": None}, "null pointer"), ({"drafts": None}, "null pointer"), ({"accepted": None}, "null pointer"),
                            ({"uniforms": None}, "uniform numbers"), ({"uniforms": None, "logits": 0}, "uniform numbers"), ({"temperature": -1.0}, "temperature"),
                            ({"temperature": math.nan}, "temperature"), ({"temperature": 1e31}, "temperature"), ({"temperature": math.inf}, "temperature"), ({"temperature": 1e-320}, "temperature"),
                            ({"temperature": 1e-307}, "temperature"), ({"space": None}, "workspace"), ({"space": 264}, "workspace"), ({"size": 127}, "workspace")):
        refused(lib, call(**change), message)
    assert lib.jq_verify_drafts(0, 0, None, 0, 0, None, None, 0, 0, None, None, 0, 3, 10, 1, 1.0, None, None, None, 0, None) == 0  # nothing to do


def test_decoder_refused(lib):
    for call in (lambda: lib.jq_decoder_set_rope(None, None, 1.0), lambda: lib.jq_decoder_set_pages(None, 4, 16, 1)):
        assert call() == _lib.JQ_ERR_INVALID


# ---- on torch tensors: nothing is called for what is refused

class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append(name)
            return 0
        return entry


@pytest.fixture()
def stub(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(paged.ops, "_front", None)
    return lib


def on_cpu(rope=None, **how):
    """A cache, a rotation and a batch whose device is the CPU's number, so that the checks behind the one of the device can be reached."""
    cache = PagedCache(8, 16, 2, 64, device=-1, k=torch.zeros(8, 2, 16, 64), v=torch.zeros(8, 2, 16, 64))
    batch = object.__new__(PagedBatch)
    batch.device, batch.prefix_length, batch._rows, batch._ahead = -1, 0, (0, 0, 4, 0, 0, 2), (None, 0, 0)
    return cache, Rope(100, 64, device=-1), batch


def rows(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("make,message", [
    (lambda: PagedBatch(rows(2, 3, dtype=I32), rows(3, dtype=I32), rows(2, dtype=I32)), "int32 CUDA tensor"), (lambda: PagedBatch([[0]], [0, 1], [1]), "int32 CUDA tensor"),
    (lambda: PagedCache(8, 16, 2, 64, k=rows(8, 2, 16, 64), v=rows(8, 2, 16, 64)), "on cuda:0 is needed"), (lambda: PagedCache(8, 16, 2, 64, k=rows(8, 2, 16, 64)), "both"),
    (lambda: PagedCache(0, 16, 2, 64), "paged cache of"), (lambda: PagedCache(8, 16, 2, 64, dtype="Q8_0"), "FP32, FP16 or BF16"), (lambda: PagedCache(8, 16, 2, 64, dtype=torch.int8), "FP32, FP16"),
    (lambda: PagedCache(8, 16, 2, 64, device=-1, k=rows(8, 2, 16, 64, dtype=F16), v=rows(8, 2, 16, 64)), "keys of a paged cache"),
    (lambda: PagedCache(8, 16, 2, 64, device=-1, k=rows(8, 2, 16, 64), v=rows(8, 16, 2, 64).transpose(1, 2)), "values of a paged cache")])
def test_construction_refused(stub, make, message):
    with pytest.raises(ValueError, match=message):
        make()
    assert stub.calls == []


@pytest.mark.parametrize("call,message", [
    (lambda r: Rope(100, 64).rotate(rows(4, 2, 64), 0), "on cpu, needed on cuda:0"), (lambda r: r.rotate(rows(4, 64), 0), "of shape"), (lambda r: r.rotate(rows(4, 2, 64).double(), 0), "FP32, FP16 or BF16"),
    (lambda r: r.rotate((rows(4, 2, 64),) * 3, 0), "3 tensors"), (lambda r: r.rotate((rows(4, 2, 64), rows(5, 2, 64)), 0), "beside"), (lambda r: r.rotate((rows(4, 2, 64), rows(4, 2, 64, dtype=F16)), 0), "beside"),
    (lambda r: r.rotate((rows(4, 2, 64), rows(4, 2, 32)), 0), "beside"), (lambda r: r.rotate(rows(4, 2, 64), rows(3, dtype=I32)), "positions"), (lambda r: r.rotate(rows(4, 2, 64), rows(4)), "positions"),
    (lambda r: r.rotate(rows(4, 2, 64), 0, out=rows(4, 2, 64, dtype=F16)), "output"), (lambda r: r.rotate(rows(4, 2, 64), 0, out=rows(4, 3, 64)), "output"),
    (lambda r: r.rotate(rows(4, 2, 64), 0, out=rows(4, 64, 2).transpose(1, 2)), "strides"), (lambda r: r.rotate(rows(4, 2, 64), 0, out=rows(1, 2, 64).expand(4, 2, 64)), "strides"),
    (lambda r: (lambda x: r.rotate(x[1:], 0, out=x[:-1]))(rows(5, 2, 64)), "overlaps"), (lambda r: (lambda x: r.rotate((x, x), 0, out=(x, x)))(rows(4, 2, 64)), "the other's output"),
    (lambda r: (lambda x, y: r.rotate((x, y), 0, out=(y, x)))(rows(4, 2, 64), rows(4, 2, 64)), "the other's output"),
    (lambda r: (lambda x, y: r.rotate((x, y), 0, out=(y, None)))(rows(4, 2, 64), rows(4, 2, 64)), "the other's output"), (lambda r: r.backward(rows(4, 2, 64), rows(4, dtype=torch.int16)), "rotation backward: positions")])
def test_rotation_refused(stub, call, message):
    rope = Rope(100, 64, device=-1)
    with pytest.raises(ValueError, match=message):
        call(rope)
    assert "jq_rope_apply" not in stub.calls


@pytest.mark.parametrize("call,message", [
    (lambda c, r, b: c.append(None, rows(3, 2, 64), rows(3, 2, 64), "b"), "PagedBatch"), (lambda c, r, b: c.append(None, rows(3, 4, 64), rows(3, 2, 64), b), "append: keys"),
    (lambda c, r, b: c.append(None, rows(3, 2, 64), rows(3, 2, 32), b), "append: values"), (lambda c, r, b: c.append(None, rows(3, 2, 64), rows(2, 2, 64), b), "append: keys"),
    (lambda c, r, b: c.append(rows(3, 8, 64, dtype=F16), rows(3, 2, 64), rows(3, 2, 64), b), "append: queries"), (lambda c, r, b: c.append(rows(2, 8, 64), rows(3, 2, 64), rows(3, 2, 64), b), "append: queries"),
    (lambda c, r, b: c.append(None, rows(3, 2, 64), rows(3, 2, 64), b, rope=Rope(10, 64)), "Rope on cuda"), (lambda c, r, b: c.append(None, rows(3, 2, 64), rows(3, 2, 64), b, rope="r"), "Rope on cuda"),
    (lambda c, r, b: c.append(rows(3, 8, 64), rows(3, 2, 64), rows(3, 2, 64), b, out=rows(3, 8, 32)), "output"),
    (lambda c, r, b: (lambda x: c.append(rows(3, 2, 64), x, rows(3, 2, 64), b, out=x))(rows(3, 2, 64)), "overlaps"),
    (lambda c, r, b: (lambda x: c.append(rows(3, 2, 64), rows(3, 2, 64), x[1:], b, out=x[:3]))(rows(4, 2, 64)), "overlaps"),
    (lambda c, r, b: c.attention(rows(3, 3, 64), b), "3 query heads on 2"), (lambda c, r, b: c.attention(rows(3, 0, 64), b), "0 query heads"), (lambda c, r, b: c.attention(rows(3, 2, 32), b), "queries of shape"),
    (lambda c, r, b: c.attention(rows(3, 2, 64).to(torch.float64), b), "FP32, FP16 or BF16"), (lambda c, r, b: (lambda x: c.attention(x, b, out=x))(rows(3, 2, 64)), "overlaps the queries"),
    (lambda c, r, b: c.attention(rows(3, 2, 64), b, out=rows(3, 2, 64, dtype=F16)), "output")])
def test_pages_refused(stub, call, message):
    cache, rope, batch = on_cpu()
    with pytest.raises(ValueError, match=message):
        call(cache, rope, batch)
    assert not {"jq_pages_append", "jq_pages_attention"} & set(stub.calls)


def test_released(stub):
    cache, rope, batch = on_cpu()
    for x in (cache, rope):
        x.release()
        x.release()
    with pytest.raises(RuntimeError, match="released"):
        rope.rotate(rows(1, 1, 64), 0)
    with pytest.raises(RuntimeError, match="released"):
        cache.attention(rows(1, 2, 64), batch)
    assert stub.calls.count("jq_rope_free") == 1 and stub.calls.count("jq_pages_free") == 1


@pytest.mark.parametrize("target", [rows(2, 4, 10), rows(4, 10), [1.0]])
def test_verification_of_host_tensors_refused(stub, target):
    with pytest.raises(ValueError, match="CUDA tensor"):
        Speculative.verify(target, rows(2, 3, dtype=I32), rows(2, 4), temperature=1.0)
    assert stub.calls == []

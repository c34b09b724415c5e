"""A pair of queries and keys of which one has no heads: what reaches the library, without a GPU, and the other's rotation, on one."""

import pytest
import torch

from jitnn_b200 import Rope, _lib, paged
from test_paged_refusals import Library


class Recorder(Library):
    def jq_rope_apply(self, h, elem, count, x, y, heads, hd, strides, *rest):
        self.calls.append(("jq_rope_apply", count, list(x), list(y), list(heads), list(strides)))
        return 0


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dims", [3, 4])
def test_the_other_is_rotated(monkeypatch, dims, inverse):
    lib = Recorder()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(paged.ops, "_front", None)
    monkeypatch.setattr(paged, "_raw_stream", lambda *a: None)
    rope = Rope(100, 64, device=-1)
    lead = (4,) if dims == 3 else (2, 4)
    full, none = torch.zeros(*lead, 3, 64), torch.zeros(*lead, 0, 64)
    strides = [0] * (dims == 3) + list(full.stride()[:-1])
    turn = rope.backward if inverse else rope.rotate
    for pair, at in (((full, none), 0), ((none, full), 1)):
        lib.calls.clear()
        got = turn(pair, 0)
        assert lib.calls == [("jq_rope_apply", 1, [full.data_ptr()], [got[at].data_ptr()], [3], strides * 2)]
        assert [x.shape for x in got] == [x.shape for x in pair]
    lib.calls.clear()
    assert [x.shape for x in turn((none, none), 0)] == [none.shape] * 2 and turn(none, 0).shape == none.shape
    assert lib.calls == []


@pytest.mark.gpu
def test_on_the_device():
    rope = Rope(100, 64)
    x = torch.randn(5, 3, 64, device="cuda")
    none = x[:, :0]
    want = rope.rotate(x, 7)
    for pair, at in (((x, none), 0), ((none, x), 1)):
        got = rope.rotate(pair, 7)
        assert torch.equal(got[at], want) and got[1 - at].shape == none.shape
    y = x.clone()
    rope.rotate((y, none), 7, out=(y, none))
    assert torch.equal(y, want)

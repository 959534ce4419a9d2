"""Calls given a stream, without a GPU: everything a call allocates and launches is inside that stream's
context, and the memory it shares with the current stream is recorded on both."""
import contextlib

import pytest

from bigrig_amd import formats as F
from bigrig_amd import layer as ops
from bigrig_amd import lib as L
from bigrig_amd.spec import E256_SHARED
from tests.helpers import small

SPEC = small(E256_SHARED, quant=F.QuantSpec(4, 32, "mxfp4"), hidden=64, inter=64, shared_inter=64, n_experts=4, top_k=2)


@pytest.fixture
def streams(monkeypatch):
    """torch's current stream as a name: `now[0]`."""
    import torch
    now = ["own"]

    @contextlib.contextmanager
    def on(s):
        was, now[0] = now[0], s
        try:
            yield
        finally:
            now[0] = was
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now[0])
    monkeypatch.setattr(ops, "_stream", lambda stream=None: now[0] if stream is None else stream)
    return now


class _Slots:
    handle = None


class _Pool:
    """Residency of `capacity` of the layer's experts, no memory behind it."""
    spec, layer, device, table_stale = SPEC, 0, _Slots(), True

    def __init__(self, capacity, seen, now):
        import numpy as np
        self.capacity, self.n_experts, self.full = capacity, SPEC.n_experts, capacity == SPEC.n_experts
        self.g2s, self.seen, self.now = np.zeros(SPEC.n_experts, int), seen, now

    def touch(self, experts, ranks=None):
        return []

    def g2s_device(self, stream):
        self.seen.append(("table", self.now[0], stream))


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
@pytest.mark.parametrize("capacity", [4, 2])
def test_the_whole_call_is_on_the_given_stream(streams, monkeypatch, activations, capacity):
    import torch
    seen = []
    sw = ops.StreamingSwitchGLU(_Pool(capacity, seen, streams), None, shared=torch.zeros(8, dtype=torch.uint8),
                                activations=activations)
    assert sw.refresh() == (capacity == 4)
    made = torch.empty

    def empty(*a, **kw):
        seen.append(("memory", streams[0], "side"))
        return made(*a, **kw)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(sw, "_forward", lambda *a, stream=None, **kw: seen.append(("forward", streams[0], stream)))
    monkeypatch.setattr(sw, "_forward_pairs", lambda *a, stream=None, **kw: seen.append(("pairs", streams[0], stream)))
    for m in (ops, __import__("bigrig_amd.mx", fromlist=["mx"])):
        monkeypatch.setattr(m, "combine", lambda *a, stream=None, **kw: seen.append(("sum", streams[0], stream)))
    idx = torch.tensor([[0, 1], [2, 3], [1, 0]], dtype=torch.int32)
    w, sg = torch.full((3, 2), 0.5), torch.ones(3)
    monkeypatch.setattr(ops, "router_topk", lambda *a: seen.append(("route", streams[0], a[-1])) or (idx, w, sg))
    monkeypatch.setattr(ops, "moe_block", lambda spec, pool, x, *a, stream=None, **kw:
                        seen.append(("block", streams[0], stream)) or x)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    moe = ops.MoELayer(SPEC, None, sw)
    for call in (lambda: sw(x, idx, stream="side"), lambda: sw.forward_combined(x, idx, w, sg, stream="side"),
                 lambda: moe(x, stream="side")):
        seen.clear()
        call()
        assert streams[0] == "own"
        kinds = {k for k, _, _ in seen}
        assert kinds & {"forward", "pairs", "block"} and "table" in kinds
        assert all(at == "side" for _, at, _ in seen), seen


def test_memory_is_recorded_on_both_streams(streams, monkeypatch):
    marks = []

    class Tensor:
        def __init__(self, name):
            self.name, self.is_cuda = name, True

        def record_stream(self, s):
            marks.append((self.name, s))
    import torch
    monkeypatch.setattr(torch, "Tensor", Tensor)
    a, b, c, out = (Tensor(n) for n in "abco")

    def call(*args):
        assert streams[0] == "side"
        return [out, None]
    got = L.on_stream("side", call, 3, a, (b, None), {"c": c})
    assert got == [out, None]
    assert marks == [("a", "side"), ("b", "side"), ("c", "side"), ("o", "own")]


def test_a_subclass_that_names_its_stream(streams, monkeypatch):
    """A block or switch whose own call passes a stream on is entered once."""
    import torch
    seen = []

    class Switch(ops.StreamingSwitchGLU):
        def __call__(self, x, indices):
            return super().__call__(x, indices, stream="side")

        def forward_combined(self, x2, idx, w, sgate=None):
            return super().forward_combined(x2, idx, w, sgate, stream="side")

    class Block(ops.MoELayer):
        def __call__(self, x):
            return super().__call__(x, stream="outer")
    sw = Switch(_Pool(4, seen, streams), None)
    assert sw.refresh()
    monkeypatch.setattr(sw, "_forward", lambda *a, **kw: seen.append(streams[0]))
    monkeypatch.setattr(ops, "router_topk", lambda *a: (idx, w, None))
    idx, w = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, 2)
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    sw(x, idx)
    sw.forward_combined(x, idx, w)
    sw.activations = "mxfp4"
    Block(SPEC, None, sw)(x)
    assert [s for s in seen if not isinstance(s, tuple)] == ["side", "side", "side"]
    assert streams[0] == "own"

"""libbrx_torch.so without a GPU: it loads beside libbrx.so, its calls are registered, and a missing one is an error."""
import os

import pytest
import torch

from bigrig_amd import lib as L
from bigrig_amd import norm as M


def test_calls_are_registered():
    ops = L.load_torch()
    assert ops is torch.ops.brx
    for name, inputs, outputs in (("enter", 4, 1), ("leave", 7, 1), ("leave_enter", 8, 2)):
        schema = getattr(ops, name).default._schema
        assert len(schema.arguments) == inputs and len(schema.returns) == outputs


def test_one_libbrx_in_the_process():
    L.load()
    L.load_torch()
    mapped = {line.split()[-1] for line in open("/proc/self/maps") if line.rstrip().endswith("libbrx.so")}
    assert mapped == {os.path.realpath(L.LIB)}


def test_a_missing_library_is_an_error(monkeypatch):
    monkeypatch.setattr(L, "_torch_ops", None)
    monkeypatch.setattr(L, "TORCH_LIB", L.TORCH_LIB + ".missing")
    with pytest.raises(RuntimeError, match="missing"):
        L.load_torch()


def test_its_errors_are_the_librarys(monkeypatch):
    def fails(*args):
        raise RuntimeError("libbrx error -2: brx_init was not called\nwhere it was raised")

    monkeypatch.setattr(M, "_with_gradients", lambda: (fails,) * 3)
    monkeypatch.setattr(M, "_on_device", lambda *t: 0)
    x = torch.zeros((2, 8), requires_grad=True)
    for call in (lambda: M.enter(x), lambda: M.leave(x, x), lambda: M.leave(x, x, next_weight=torch.ones(8))):
        with pytest.raises(L.BrxError, match="brx_init") as e:
            call()
        assert e.value.code == L.BRX_ESTATE

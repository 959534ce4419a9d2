"""Forward-mode derivatives and recorders of torch's operations met by the operators around a block's experts: neither gets a
sum or a program that silently lacks a call. On the CPU; the launches are replaced by writes that torch does not see either."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from bigrig_amd import dispatch as D
from bigrig_amd import grouped as G
from bigrig_amd import lib as L
from bigrig_amd import norm as M

T, K, H, E = 3, 2, 8, 4
B = torch.bfloat16
SEED = torch.Generator().manual_seed(1)


class Launches:
    """A library whose calls are counted and write to their output."""
    calls = 0

    def write(self, out, n):
        self.calls += 1
        C.memset(out, 0, n)
        return 0

    def brx_pairs_dispatch(self, x, x_row, position, T, k, H, dtype, rows, stream):
        return self.write(rows, 4 * T * k * H)

    def brx_pairs_combine(self, rows, w, position, T, k, H, dtype, out, stream):
        return self.write(out, 4 * T * H)

    def brx_norm_forward(self, y, y_row, y_dtype, r, r_row, r_dtype, post, post_dtype, gate, form, gate_dtype, nxt, next_dtype, scale,
                         eps, T, H, new, h, rstd_y, rstd_n, stream):
        return self.write(h, 4 * T * H)

    def brx_grouped_product(self, rows, weight, w_expert, w_row, bias, offsets, P, E, K, N, dtype, out, stream):
        return self.write(out, 2 * P * N)


@pytest.fixture
def lib(monkeypatch):
    got = Launches()
    monkeypatch.setattr(L, "load", lambda path=None: got)
    for m in (D, G, M):
        monkeypatch.setattr(m, "_on_device", lambda *t: -1)
        monkeypatch.setattr(m, "_handle", lambda d: 0)
    return got


def plan():
    return D.Dispatch(torch.arange(T * K, dtype=torch.int32), torch.arange(T * K, dtype=torch.int32).view(T, K),
                      torch.tensor([0, 1, 2, 3, T * K], dtype=torch.int32))


def cases():
    """(call, the tensors it would follow)."""
    p = plan()
    rows, w = torch.randn((T * K, H), generator=SEED), torch.rand((T, K), generator=SEED)
    x16, m16 = torch.randn((T * K, H), generator=SEED).to(B), torch.randn((E, H, H), generator=SEED).to(B)
    b16 = torch.randn((E, H), generator=SEED).to(B)
    return {"dispatch": (lambda x: D.dispatch(x, p), [torch.randn((T, H), generator=SEED)]),
            "combine": (lambda r, s: D.combine(r, p, s), [rows, w]),
            "sum": (lambda r: D.combine(r, p), [rows]),
            "enter": (lambda x, v: M.enter(x, v), [torch.randn((T, H), generator=SEED), torch.rand(H, generator=SEED)]),
            "leave": (lambda *t: M.leave(*t[:4], 0.5, t[4])[1], [torch.randn((T, H), generator=SEED) for _ in range(2)]
                      + [torch.rand(n, generator=SEED) for n in (H, (T, 1), H)]),
            "product": (lambda r, m, b: G.product(r, m, p.offsets, b), [x16, m16, b16])}


@pytest.mark.parametrize("name", ["dispatch", "combine", "sum", "enter", "leave", "product"])
def test_a_tangent_is_refused(lib, name):
    call, ts = cases()[name]
    want = call(*ts)
    with fw.dual_level():
        # (no tangent among them: the call as it is)
        assert call(*ts).shape == want.shape
        for i in range(len(ts)):
            for on in (True, False):      # torch follows tangents under no_grad, too
                dual = [fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ts)]
                with torch.set_grad_enabled(on), pytest.raises(RuntimeError, match="tangent"):
                    call(*dual)
    assert call(*ts).shape == want.shape


@pytest.mark.parametrize("name", ["dispatch", "combine", "sum", "product"])
def test_a_gradient_with_a_tangent_is_refused(lib, name):
    call, ts = cases()[name]
    ts = [t.requires_grad_() for t in ts]
    with fw.dual_level():
        out = call(*ts)
        d = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(out, ts, d)


@pytest.mark.parametrize("record", [lambda f, *t: torch.jit.trace(f, t, check_trace=False), lambda f, *t: make_fx(f)(*t)])
@pytest.mark.parametrize("name", ["dispatch", "combine", "sum", "enter", "leave", "product"])
def test_a_recorder_is_refused(lib, name, record):
    call, ts = cases()[name]
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="recorded"):
            record(lambda *t: call(*t) * 2, *(t.detach().requires_grad_(grad) for t in ts))
    with pytest.raises(RuntimeError, match="recorded"):
        record(lambda i: D.plan(i, E).order * 2, torch.zeros((T, K), dtype=torch.int32))
    assert lib.calls == 0
    call(*ts)                             # (outside, the call as it is)

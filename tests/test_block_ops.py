"""The operators around a block's experts without a GPU: what they refuse, in Python and at the C-ABI, before anything is
launched."""
import ctypes as C

import pytest
import torch

from bigrig_amd import dispatch as D
from bigrig_amd import grouped as G
from bigrig_amd import lib as L
from bigrig_amd import norm as M
from bigrig_amd.layered import MoEWeights, prefill

B, F, S = torch.bfloat16, torch.float16, torch.float32
I = torch.int32


def meta(*shape, dtype=B):
    """A tensor of a size that is never allocated."""
    return torch.empty(shape, dtype=dtype, device="meta")


def plan(T=4, k=2, E=3):
    return D.Dispatch(torch.zeros(T * k, dtype=I), torch.zeros((T, k), dtype=I), torch.zeros(E + 1, dtype=I))


@pytest.mark.parametrize("idx,E,what", [
    (torch.zeros((4, 2), dtype=torch.int64), 4, "int32"), (torch.zeros(8, dtype=I), 4, "T, k"),
    (torch.zeros((4, 2), dtype=I), 0, "experts"), (torch.zeros((4, 2), dtype=I), 513, "experts"),
    (torch.zeros((4, 0), dtype=I), 4, "a token"), (torch.zeros((1, 65), dtype=I), 128, "a token"),
    (meta(1 << 20, 9, dtype=I), 16, "pairs"), (torch.zeros((4, 2), dtype=I), 4, "GPU")])
def test_plan_refuses(idx, E, what):
    with pytest.raises(ValueError, match=what):
        D.plan(idx, E)


@pytest.mark.parametrize("x,p,what", [
    (torch.zeros((4, 8), dtype=torch.int32), plan(), "float32"), (torch.zeros((5, 8)), plan(), "4 tokens"),
    (torch.zeros((4, 2, 8)), plan(), "4 tokens"), (torch.zeros((4, 8193)), plan(), "8192"), (torch.zeros((4, 0)), plan(), "values"),
    (torch.zeros((4, 8)), plan(), "GPU"),
    (torch.zeros((4, 8)), plan()._replace(position=torch.zeros((4, 2))), "int32"),
    (torch.zeros((4, 8)), plan()._replace(position=torch.zeros((2, 4), dtype=I).t()), "contiguous"),
    (meta(1 << 20, 8), plan()._replace(position=meta(1 << 20, 9, dtype=I)), "at most")])
def test_dispatch_refuses(x, p, what):
    with pytest.raises(ValueError, match=what):
        D.dispatch(x, p)


@pytest.mark.parametrize("rows,w,what", [
    (torch.zeros((8, 8), dtype=torch.float64), None, "float32"), (torch.zeros((7, 8)), None, "8 rows"),
    (torch.zeros((4, 2, 8)), None, "8 rows"), (torch.zeros((8, 8)), torch.zeros((4, 2), dtype=B), "float32"),
    (torch.zeros((8, 8)), torch.zeros(8), "w must"), (torch.zeros((8, 8200)), None, "8192"), (torch.zeros((8, 8)), None, "GPU")])
def test_combine_refuses(rows, w, what):
    with pytest.raises(ValueError, match=what):
        D.combine(rows, plan(), w)


def off(E):
    return torch.zeros(E + 1, dtype=I)


@pytest.mark.parametrize("rows,weight,offsets,bias,what", [
    (torch.zeros((4, 8)), torch.zeros((2, 8, 8)), off(2), None, "bfloat16 or float16"),
    (meta(4, 8), meta(2, 8, 8, dtype=F), off(2), None, "one type"),
    (meta(4, 8), meta(2, 8, 8), off(2), meta(2, 8, dtype=F), "one type"),
    (meta(4, 16), meta(2, 8, 8), off(2), None, "E, N, K"), (meta(4, 8), meta(8, 8), off(2), None, "E, N, K"),
    (meta(4, 12), meta(2, 8, 12), off(2), None, "multiple of 8"), (meta(4, 8), meta(2, 20, 8), off(2), None, "multiple of 8"),
    (meta(4, 8), meta(2, 8200, 8), off(2), None, "8192"), (meta(4, 8), meta(0, 8, 8), off(0), None, "experts"),
    (meta(4, 8), meta(513, 8, 8), off(513), None, "experts"), (meta((1 << 23) + 1, 8), meta(2, 8, 8), off(2), None, "rows"),
    (meta(4, 8), meta(2, 8, 8), off(3), None, "offsets"), (meta(4, 8), meta(2, 8, 8), off(2).long(), None, "offsets"),
    (meta(4, 8), meta(2, 8, 8), off(2), meta(2, 16), "bias"),
    (meta(4, 8), meta(2, 8, 8).transpose(1, 2), off(2), None, "contiguous"),
    (torch.zeros((4, 8), dtype=B), torch.zeros((2, 8, 12), dtype=B)[:, :, :8], off(2), None, "strides"),
    (torch.zeros((4, 8), dtype=B), torch.zeros((2, 8, 8), dtype=B), off(2), None, "GPU")])
def test_product_refuses(rows, weight, offsets, bias, what):
    with pytest.raises(ValueError, match=what):
        G.product(rows, weight, offsets, bias)


@pytest.mark.parametrize("x,kw,what", [
    (torch.zeros((4, 8), dtype=torch.float64), {}, "float32"), (torch.zeros((4, 8), dtype=B), dict(dtype=F), "own type"),
    (torch.zeros((4, 8), dtype=B), dict(dtype=S), "own type"), (torch.zeros(()), {}, "dimensions"),
    (torch.zeros((4, 8200)), {}, "8192"), (torch.zeros((4, 0)), {}, "values"), (torch.zeros((4, 8)), dict(eps=0.0), "eps"),
    (torch.zeros((4, 8)), dict(eps=float("nan")), "eps"), (torch.zeros((4, 8)), dict(weight=torch.zeros(7)), "weight"),
    (torch.zeros((4, 8)), dict(weight=torch.zeros(8, dtype=I)), "weight"), (meta((1 << 23) + 1, 8), {}, "rows"),
    (torch.zeros((4, 8)), {}, "GPU")])
def test_enter_refuses(x, kw, what):
    with pytest.raises(ValueError, match=what):
        M.enter(x, **kw)


@pytest.mark.parametrize("y,r,kw,what", [
    (torch.zeros((4, 8), dtype=B), torch.zeros((4, 8), dtype=F), {}, "residual"),
    (torch.zeros((4, 8)), torch.zeros((4, 8), dtype=B), {}, "residual"), (torch.zeros((4, 8)), torch.zeros((2, 2, 8)), {}, "one shape"),
    (torch.zeros((4, 8)), torch.zeros((4, 8)), dict(gate=torch.zeros(4)), "gate"),
    (torch.zeros((4, 8)), torch.zeros((4, 8)), dict(gate=torch.zeros((1, 8))), "gate"),
    (torch.zeros((4, 8)), torch.zeros((4, 8)), dict(gate=torch.zeros(8, dtype=I)), "gate"),
    (torch.zeros((4, 8)), torch.zeros((4, 8)), dict(weight=torch.zeros((1, 8))), "weight"),
    (torch.zeros((4, 8)), torch.zeros((4, 8)), dict(next_weight=torch.zeros(9)), "next_weight"),
    (torch.zeros((4, 8)), torch.zeros((4, 8)), dict(eps=-1.0), "eps"), (torch.zeros((4, 8)), torch.zeros((4, 8)), {}, "GPU")])
def test_leave_refuses(y, r, kw, what):
    with pytest.raises(ValueError, match=what):
        M.leave(y, r, **kw)


def test_prefill_refuses_norms_without_a_residual_sum():
    with pytest.raises(ValueError, match="residual"):
        prefill(None, [MoEWeights(0, None, norms=M.BlockNorms())], None, [], None, residual=False)


def test_prefill_refuses_other_types_through_a_block_without_norms():
    with pytest.raises(ValueError, match="bfloat16"):
        prefill(None, [MoEWeights(0, None, norms=M.BlockNorms()), MoEWeights(1, None)], None, [torch.zeros((2, 8))], None)


# ------------------------------------------------------------------ the C-ABI
def call(name, *args):
    rc = getattr(L.load(), name)(*args)
    return rc, L.load().brx_last_error().decode()


def test_workspace_sizes():
    out = C.c_size_t()
    lib = L.load()
    for n, E, want in ((0, 4, 0), (16384, 512, 0), (16385, 4, 5 * 5 * 4), (1 << 23, 512, 512 * 513 * 4)):
        L.check(lib.brx_pairs_workspace_bytes(n, E, C.byref(out)))
        assert out.value == want, (n, E)
    for bad in ((-1, 4), ((1 << 23) + 1, 4), (8, 0), (8, 513)):
        assert lib.brx_pairs_workspace_bytes(*bad, C.byref(out)) == L.BRX_EINVAL
    assert lib.brx_pairs_workspace_bytes(8, 4, None) == L.BRX_EINVAL
    L.check(lib.brx_norm_workspace_bytes(7, 100, C.byref(out)))
    assert out.value >= 3 * 100 * 4
    for bad in ((-1, 8), (4, 0), (4, 8193), ((1 << 23) + 1, 8)):
        assert lib.brx_norm_workspace_bytes(*bad, C.byref(out)) == L.BRX_EINVAL


def ptr(n=4096):
    """Host memory that is never touched: the calls below are refused before a launch."""
    buf = C.create_string_buffer(n + 32)
    ptr.keep = getattr(ptr, "keep", []) + [buf]
    return (C.addressof(buf) + 31) & ~31


def test_c_calls_check_their_arguments():
    p = ptr()
    bad = [
        ("brx_pairs_plan", p, -1, 2, 4, p, p, p, None, 0, None), ("brx_pairs_plan", p, 4, 0, 4, p, p, p, None, 0, None),
        ("brx_pairs_plan", p, 4, 65, 4, p, p, p, None, 0, None), ("brx_pairs_plan", p, 4, 2, 0, p, p, p, None, 0, None),
        ("brx_pairs_plan", p, 4, 2, 513, p, p, p, None, 0, None), ("brx_pairs_plan", p, 1 << 23, 2, 4, p, p, p, None, 0, None),
        ("brx_pairs_dispatch", p, 8, p, -1, 2, 8, 1, p, None), ("brx_pairs_dispatch", p, 8, p, 4, 2, 0, 1, p, None),
        ("brx_pairs_dispatch", p, 8, p, 4, 2, 8193, 1, p, None), ("brx_pairs_dispatch", p, 8, p, 4, 2, 8, 3, p, None),
        ("brx_pairs_combine", p, p, p, 4, 65, 8, 1, p, None), ("brx_pairs_combine", p, p, p, 1 << 23, 2, 8, 1, p, None),
        ("brx_pairs_combine_backward", p, 8, p, p, p, 4, 2, 8, -1, p, p, None),
        ("brx_grouped_product", p, p, 64, 8, None, p, -1, 2, 8, 8, 1, p, None),
        ("brx_grouped_product", p, p, 64, 8, None, p, 4, 0, 8, 8, 1, p, None),
        ("brx_grouped_product", p, p, 64, 8, None, p, 4, 2, 12, 8, 1, p, None),
        ("brx_grouped_product", p, p, 64, 8, None, p, 4, 2, 8, 8200, 1, p, None),
        ("brx_grouped_product", p, p, 64, 8, None, p, 4, 2, 8, 8, 0, p, None),
        ("brx_grouped_product_backward", p, p, p, 64, 8, p, (1 << 23) + 1, 2, 8, 8, 1, p, p, p, None),
        ("brx_grouped_product_backward", p, p, p, 64, 8, p, 4, 513, 8, 8, 1, p, p, p, None),
        ("brx_norm_forward", p, 8, 0, p, 8, 1, None, 0, None, 0, 0, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 5, p, 8, 5, None, 0, None, 0, 0, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, None, 0, None, 0, 0, None, 0, 1.0, 1e-6, 4, 8193, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, None, 0, None, 0, 0, None, 0, 1.0, 1e-6, -4, 8, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, None, 0, p, 0, 1, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, None, 0, None, 2, 1, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, None, 0, p, 4, 1, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, p, 7, None, 0, 0, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_forward", None, 8, 1, p, 8, 1, p, 1, None, 0, 0, None, 0, 1.0, 1e-6, 4, 8, None, p, None, None, None),
    ]
    for name, *args in bad:
        rc, msg = call(name, *args)
        assert rc == L.BRX_EINVAL and msg, (name, args, rc)


def test_c_calls_need_a_device_first():
    # valid arguments without brx_init: refused before any memory is read (this process has no GPU)
    if torch.cuda.is_available():
        pytest.skip("brx_init may have been called")
    p = ptr()
    good = [
        ("brx_pairs_plan", p, 4, 2, 4, p, p, p, None, 0, None), ("brx_pairs_dispatch", p, 8, p, 4, 2, 8, 1, p, None),
        ("brx_pairs_combine", p, p, p, 4, 2, 8, 1, p, None),
        ("brx_pairs_combine_backward", p, 8, p, p, p, 4, 2, 8, 1, p, p, None),
        ("brx_grouped_product", p, p, 64, 8, None, p, 4, 2, 8, 8, 1, p, None),
        ("brx_grouped_product_backward", p, p, p, 64, 8, p, 4, 2, 8, 8, 1, p, p, p, None),
        ("brx_norm_forward", p, 8, 1, p, 8, 1, None, 0, None, 0, 0, None, 0, 1.0, 1e-6, 4, 8, p, None, None, None, None),
        ("brx_norm_backward", p, 8, 1, p, 8, 1, None, 0, None, 0, 0, None, 0, 1.0, 4, 8, None, None, p, None, p, p, None, None,
         None, None, 0, None),
    ]
    for name, *args in good:
        rc, msg = call(name, *args)
        assert rc == L.BRX_ESTATE, (name, rc, msg)

"""Tokens sorted by expert and back, with the routing's weights, and the gradients, on libbrx.

The reference sorts a chunk's (token, expert) pairs on the host and puts the experts' rows back by
indexing (bigrig_engine/stream.py:1526-1530, 1558-1561); the layer forms here (`layer.moe_forward`) do both
inside their kernels. These are the steps by themselves, for experts that are a program's own -- trained
ones (`grouped.product`), another library's, another device's:

* `plan`: which row each pair takes, the rows of one expert after another's;
* `dispatch`: the tokens' rows in that order;
* `combine`: the sum of each token's rows, times the routing's weights.

A pair of an expert outside [0, n_experts) -- padding, another device's expert: -1 -- is dropped: no row is its own,
`combine` leaves it out, its gradients are 0. The rows behind the last pair's are 0.

`dispatch` and `combine` have gradients (taken once: create_graph=True is refused). Sums are float32, over a
token's pairs in their order, rounded once, and every result is the same bits on every run. Tensors live on
the current device; scratch is allocated per call by torch, on the call's stream. Given a `stream`, the whole call
runs there (and its gradient): the inputs have to be ready on it. A gradient that is captured into a graph is taken of
leaves that no eager graph holds meanwhile (`detach().requires_grad_()` inside the capture): torch ends the process
where an eager graph's leaf on another stream is met in a capture.

There are no forward-mode derivatives: a tensor with a tangent is refused. So are the calls where torch's operations are
recorded (`torch.jit.trace`, make_fx): the recorded program would not hold them.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import lib as L
from .mx import _handle, _on_device

MAX_PAIRS = 1 << 23     # (token, expert) pairs of one call
MAX_EXPERTS = 512
MAX_TOP_K = 64
MAX_WIDTH = 8192        # values of a row


class Dispatch(NamedTuple):
    """`order` int32 [T k]: the pair (t k + j) in each row, -1 behind the last; `position` int32 [T, k]: the row of
    each pair, negative where it is dropped (-1 - one of the rows behind the last, a different one for each);
    `offsets` int32 [E + 1]: where each expert's rows start, the last entry the pairs that were kept."""
    order: object
    position: object
    offsets: object


_TYPES = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def _dtype(t, what: str) -> int:
    dt = _TYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{what} is {t.dtype}: float32, bfloat16 or float16")
    return dt


_is_tracing = torch._C._is_tracing
_modes = torch._C._len_torch_dispatch_stack


def _refuse_recorders() -> None:
    """A recorder of torch's operations (`torch.jit.trace`, make_fx) sees a launch's allocations only: its program would read
    memory that nothing wrote. (A trace would hold an autograd function, but not the checks of shapes before it.)"""
    if _is_tracing() or (_modes() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None):
        raise RuntimeError("torch's operations are being recorded: a recorded program would not hold this call")


def _refuse_tangents(tensors) -> None:
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("a tensor with a tangent: there are no forward-mode derivatives")


def _recorded(*tensors) -> bool:
    """Whether a gradient is recorded of a call. It is refused where its result would silently lack a derivative or a
    program the call."""
    if _is_tracing() or _modes():
        _refuse_recorders()
    if forward_ad._current_level >= 0:
        _refuse_tangents(tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


@functools.lru_cache(maxsize=1024)
def _plan_bytes(n: int, E: int) -> int:
    out = C.c_size_t()
    L.check(L.load().brx_pairs_workspace_bytes(n, E, C.byref(out)))
    return out.value


def plan(idx, n_experts: int, stream=None) -> Dispatch:
    """The plan of a routing idx [T, k] (int32, as `layer.router_topk` returns it) of n_experts experts: a stable sort of
    its pairs by expert. It is made once for a routing, whatever is sent through it."""
    if stream is not None:
        return L.on_stream(stream, plan, idx, n_experts)
    if idx.dtype != torch.int32 or idx.dim() != 2:
        raise ValueError(f"idx must be int32 [T, k], got {idx.dtype} {tuple(idx.shape)}")
    T, k = idx.shape
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"{n_experts} experts outside [1, {MAX_EXPERTS}]")
    if not 1 <= k <= MAX_TOP_K:
        raise ValueError(f"{k} experts a token outside [1, {MAX_TOP_K}]")
    n = T * k
    if n > MAX_PAIRS:
        raise ValueError(f"{n} pairs in one call: at most {MAX_PAIRS}")
    _refuse_recorders()
    device = _on_device(idx)
    if not idx.is_contiguous():
        idx = idx.contiguous()
    order = idx.new_empty(n)
    position = idx.new_empty((T, k))
    offsets = idx.new_empty(n_experts + 1)
    need = _plan_bytes(n, n_experts)
    ws = idx.new_empty(need // 4) if need else None
    rc = L.load().brx_pairs_plan(idx.data_ptr(), T, k, n_experts, order.data_ptr(), position.data_ptr(),
                                 offsets.data_ptr(), None if ws is None else ws.data_ptr(), need, _handle(device))
    if rc:
        L.check(rc)
    return Dispatch(order, position, offsets)


def _position(plan: Dispatch):
    p = plan.position
    if p.dtype != torch.int32 or p.dim() != 2 or not p.is_contiguous():
        raise ValueError(f"the plan's position must be contiguous int32 [T, k], got {p.dtype} {tuple(p.shape)}")
    T, k = p.shape
    if not 1 <= k <= MAX_TOP_K or T * k > MAX_PAIRS:
        raise ValueError(f"a plan of {T} x {k} pairs: 1 to {MAX_TOP_K} a token, at most {MAX_PAIRS}")
    return p, T, k


def _width(H: int) -> None:
    if not 1 <= H <= MAX_WIDTH:
        raise ValueError(f"rows of {H} values: 1 to {MAX_WIDTH}")


def _gather(x, position, T: int, k: int):
    """rows[position[t, j]] = x[t]; x [T, H], rows strided."""
    device = _on_device(x, position)
    H = x.shape[1]
    rows = x.new_empty((T * k, H))
    rc = L.load().brx_pairs_dispatch(x.data_ptr(), x.stride(0) if T > 1 else H, position.data_ptr(), T, k, H,
                                     _TYPES[x.dtype], rows.data_ptr(), _handle(device))
    if rc:
        L.check(rc)
    return rows


def _sum(rows, w, position, T: int, k: int):
    device = _on_device(rows, w, position)
    H = rows.shape[1]
    out = rows.new_empty((T, H))
    rc = L.load().brx_pairs_combine(rows.data_ptr(), None if w is None else w.data_ptr(), position.data_ptr(), T, k, H,
                                    _TYPES[rows.dtype], out.data_ptr(), _handle(device))
    if rc:
        L.check(rc)
    return out


def _strided(x):
    """x [T, H] with contiguous rows, in place where they are."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _once(backward):
    """A gradient that has none itself. Asked for one that could be differentiated again (create_graph=True), it is
    refused: torch would take it for a constant wherever the gradient given does not ask for one."""
    @functools.wraps(backward)
    def call(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError("this gradient is taken once: create_graph=True is refused")
        if forward_ad._current_level >= 0:
            _refuse_tangents(grads)
        return backward(ctx, *grads)
    return call


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, T, k):
        ctx.save_for_backward(position)
        ctx.sizes = T, k
        return _gather(x, position, T, k)

    @staticmethod
    @_once
    def backward(ctx, drows):
        position, = ctx.saved_tensors
        return _sum(drows.contiguous(), None, position, *ctx.sizes), None, None, None


def dispatch(x, plan: Dispatch, stream=None):
    """Rows [T k, H] of tokens x [T, H] (float32, bfloat16 or float16; rows may be strided) in the plan's order: row r is
    the token of pair order[r]. Its gradient is the sum of a token's rows."""
    if stream is not None:
        return L.on_stream(stream, dispatch, x, plan)
    position, T, k = _position(plan)
    _dtype(x, "x")
    if x.dim() != 2 or x.shape[0] != T:
        raise ValueError(f"x {tuple(x.shape)}: the plan is of {T} tokens")
    _width(x.shape[1])
    x = _strided(x)
    if _recorded(x):
        return _Dispatch.apply(x, position, T, k)
    return _gather(x, position, T, k)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, w, position, T, k):
        need = ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if need else None, w, position)
        ctx.sizes = T, k, rows.shape[1]
        return _sum(rows, w, position, T, k)

    @staticmethod
    @_once
    def backward(ctx, dout):
        rows, w, position = ctx.saved_tensors
        T, k, H = ctx.sizes
        dout = _strided(dout)
        drows = dout.new_empty((T * k, H)) if ctx.needs_input_grad[0] else None
        dw = w.new_empty((T, k)) if ctx.needs_input_grad[1] else None
        ptr = L.ptr
        rc = L.load().brx_pairs_combine_backward(
            dout.data_ptr(), dout.stride(0) if T > 1 else H, ptr(rows), ptr(w), position.data_ptr(), T, k, H,
            _TYPES[dout.dtype], ptr(drows), ptr(dw), _handle(dout.get_device()))
        if rc:
            L.check(rc)
        return drows, dw, None, None, None


def combine(rows, plan: Dispatch, w=None, stream=None):
    """out [T, H] = sum_j w[t, j] rows[position[t, j]] over the pairs that were kept: the experts' rows [T k, H] (float32,
    bfloat16 or float16) back at their tokens, times the routing's weights w [T, k] (float32; None: ones). Gradients
    of rows and w."""
    if stream is not None:
        return L.on_stream(stream, combine, rows, plan, w)
    position, T, k = _position(plan)
    _dtype(rows, "rows")
    if rows.dim() != 2 or rows.shape[0] != T * k:
        raise ValueError(f"rows {tuple(rows.shape)}: the plan has {T * k} rows")
    _width(rows.shape[1])
    if w is not None and (w.dtype != torch.float32 or w.shape != (T, k)):
        raise ValueError(f"w must be float32 [{T}, {k}], got {w.dtype} {tuple(w.shape)}")
    rows = rows.contiguous()
    if w is not None:
        w = w.contiguous()
    if _recorded(rows, w):
        return _Combine.apply(rows, w, position, T, k)
    return _sum(rows, w, position, T, k)

"""Norms at both ends of a block, fused with its gate, residual scale and residual sum, and their gradients.

With n(v; w) = v / sqrt(mean(v^2) + eps) * w (root mean square, over the last dimension):

* `enter`: h = n(x; weight), what a block reads;
* `leave`: u = n(y; weight) (or y), new = residual + scale * gate * u and, given the next block's weights,
  h = n(new; next_weight), in one pass over the block's result y and the residual stream.

`new` is rounded to the residual's type and h made of what was rounded, so `leave` with next_weight gives the
bits that `leave` and `enter` give one after the other. Statistics and sums are float32, each result rounded once.
Gradients are taken once (create_graph=True is refused) and are the same bits on every run. Streams, tangents and recorders as
in `dispatch`. The reference leaves norms and residual sums to MLX (bigrig_engine/layered.py:110-121 calls a whole
decoder layer).

`BlockNorms` puts both around a block of `layer.MoELayer` or `layered.prefill`.
"""
from __future__ import annotations

import functools
import re
from dataclasses import dataclass

import torch

from . import lib as L
from .dispatch import MAX_PAIRS as MAX_ROWS
from .dispatch import _TYPES, _dtype, _recorded, _width
from .mx import _handle, _on_device

EPS = 1e-6
_NO_GATE, _CHANNEL, _ROW, _FULL = 0, 1, 2, 3
_ENTER, _LEAVE, _LEAVE_ENTER = 0, 1, 2
_ERROR = re.compile(r"libbrx error (-?\d+): (.*)")


@dataclass
class BlockNorms:
    """x -> x + scale * gate * n(block(n(x; pre)); post): the norms, gate [H] and residual scale of a block (tensors on
    the GPU; pre None: a norm without weights, post None: no norm, gate None: ones). The residual stream x is bfloat16
    or float32, the block's tensors bfloat16. (The library's blocks have no gradient, so none is recorded.)"""
    pre: object = None
    post: object = None
    gate: object = None
    scale: float = 1.0
    eps: float = EPS

    def enter(self, x):
        """What the block reads of the residual stream x."""
        with torch.no_grad():
            return enter(x, self.pre, self.eps, torch.bfloat16)

    def leave(self, y, x, after: BlockNorms | None = None):
        """(the residual stream behind the block, what the next block reads of it), given the next block's norms; the
        second is None where these need a pass of their own."""
        with torch.no_grad():
            if after is not None and after.pre is not None and after.eps == self.eps:
                return leave(y, x, self.post, self.gate, self.scale, after.pre, self.eps)
            return leave(y, x, self.post, self.gate, self.scale, eps=self.eps), None

    def around(self, block, x):
        """The residual stream x [T, H] behind `block`, a call from [T, H] to [T, H]."""
        return self.leave(block(self.enter(x)), x)[0]


@functools.cache
def _with_gradients():
    """The calls that record a gradient (csrc/brx_torch.cpp): (enter, leave, leave and enter). (The functions under torch's
    operators: torch.compile breaks its graph at them, where it would run the operators on tensors without memory.)"""
    ops = L.load_torch()
    return ops.enter.default._op, ops.leave.default._op, ops.leave_enter.default._op


def _record(call: int, *args):
    try:
        return _with_gradients()[call](*args)
    except RuntimeError as e:
        found = _ERROR.match(str(e))
        if found is None:
            raise
        raise L.BrxError(int(found[1]), found[2]) from None


def _vector(t, H: int, what: str):
    """A weight [H] of any of the three types."""
    _dtype(t, what)
    if t.shape != (H,):
        raise ValueError(f"{what} {tuple(t.shape)}, the rows have {H} values")
    return t.contiguous()


def _rows(t, H: int):
    """t [..., H] as rows [T, H], in place where they are evenly strided."""
    t2 = t if t.dim() == 2 else t.reshape(-1, H)
    return t2 if t2.stride(1) == 1 or H == 1 else t2.contiguous()


def _gate_form(gate, shape) -> int:
    if gate is None:
        return _NO_GATE
    _dtype(gate, "gate")
    if tuple(gate.shape) == (shape[-1],):
        return _CHANNEL
    if tuple(gate.shape) == (*shape[:-1], 1):
        return _ROW
    if tuple(gate.shape) == tuple(shape):
        return _FULL
    raise ValueError(f"gate {tuple(gate.shape)}: one value a channel {(shape[-1],)}, a row {(*shape[:-1], 1)} or an element "
                     f"{tuple(shape)}")


def _type(t) -> int:
    return 0 if t is None else _TYPES[t.dtype]


def _stride(t, T: int, H: int) -> int:
    return t.stride(0) if T > 1 else H


def _forward(y, r, post, gate, form, nxt, scale, eps, make_h, h_type):
    """(new_r or None, h or None) of rows r [T, H] and, for `leave`, y [T, H]; no gradient is recorded."""
    device = _on_device(y, r, post, gate, nxt)
    T, H = r.shape
    new = None if y is None else r.new_empty((T, H))
    h = r.new_empty((T, H), dtype=h_type) if make_h else None
    ptr = L.ptr
    L.check(L.load().brx_norm_forward(
        ptr(y), 0 if y is None else _stride(y, T, H), _TYPES[h_type], r.data_ptr(), _stride(r, T, H), _TYPES[r.dtype],
        ptr(post), _type(post), ptr(gate), form, _type(gate), ptr(nxt), _type(nxt), scale, eps, T, H, ptr(new), ptr(h),
        None, None, _handle(device)))
    return new, h


def _check_count(T: int) -> None:
    if T > MAX_ROWS:
        raise ValueError(f"{T} rows in one call: at most {MAX_ROWS}")


def _check_eps(eps: float) -> None:
    if not 1.17549435e-38 <= eps < 3.4e38:
        raise ValueError(f"eps {eps} must be a positive, normal float32 value")


def enter(x, weight=None, eps: float = EPS, dtype=None, stream=None):
    """n(x; weight) of x [..., H] (float32, bfloat16 or float16; H up to 8192; rows may be strided), in `dtype`: x's, or any
    of the three for a float32 x. weight [H] (any of the three; None: ones). Gradients of x and weight."""
    if stream is not None:
        return L.on_stream(stream, enter, x, weight, eps, dtype)
    _dtype(x, "x")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _TYPES or (dtype != x.dtype and x.dtype != torch.float32):
        raise ValueError(f"a norm of {x.dtype} in {dtype}: in its own type, or from float32")
    if x.dim() == 0:
        raise ValueError("x has no dimensions")
    H = x.shape[-1]
    _width(H)
    _check_eps(eps)
    if weight is not None:
        weight = _vector(weight, H, "weight")
    x2 = _rows(x, H)
    _check_count(x2.shape[0])
    if _recorded(x2, weight):
        _on_device(x2, weight)
        h = _record(_ENTER, x2, weight, eps, dtype)
    else:
        h = _forward(None, x2, None, None, _NO_GATE, weight, 1.0, eps, True, dtype)[1]
    return h if h.shape == x.shape else h.view(x.shape)


def leave(y, residual, weight=None, gate=None, scale: float = 1.0, next_weight=None, eps: float = EPS, stream=None):
    """new = residual + scale * gate * n(y; weight) of a block's result y [..., H] (float32, bfloat16 or float16; weight None:
    y as it is) and the residual stream (y's type, or float32), in the residual's type. gate: one value a channel [H],
    a row [..., 1] or an element [..., H] (None: ones). With next_weight [H]: (new, n(new; next_weight) in y's type).
    Weights and gate of any of the three types. Rows may be strided. Gradients of all tensors given."""
    if stream is not None:
        return L.on_stream(stream, leave, y, residual, weight, gate, scale, next_weight, eps)
    _dtype(y, "y")
    if residual.dtype != y.dtype and residual.dtype != torch.float32:
        raise ValueError(f"a residual of {residual.dtype} with y of {y.dtype}: the same, or float32")
    if y.dim() == 0 or y.shape != residual.shape:
        raise ValueError(f"y {tuple(y.shape)} and residual {tuple(residual.shape)} must be of one shape [..., H]")
    H = y.shape[-1]
    _width(H)
    _check_eps(eps)
    scale = float(scale)
    form = _gate_form(gate, y.shape)
    if gate is not None:
        gate = gate.contiguous()
    if weight is not None:
        weight = _vector(weight, H, "weight")
    make_h = next_weight is not None
    if make_h:
        next_weight = _vector(next_weight, H, "next_weight")
    y2, r2 = _rows(y, H), _rows(residual, H)
    _check_count(y2.shape[0])
    if _recorded(y2, r2, weight, gate, next_weight):
        _on_device(y2, r2, weight, gate, next_weight)
        if make_h:
            new, h = _record(_LEAVE_ENTER, y2, r2, weight, gate, form, scale, next_weight, eps)
        else:
            new, h = _record(_LEAVE, y2, r2, weight, gate, form, scale, eps), None
    else:
        new, h = _forward(y2, r2, weight, gate, form, next_weight, scale, eps, make_h, y.dtype)
    if new.shape != y.shape:
        new, h = new.view(y.shape), None if h is None else h.view(y.shape)
    return (new, h) if make_h else new

"""Products of rows sorted by expert with each expert's matrix, and their gradients, on libbrx.

The reference multiplies sorted rows by quantised experts (`mx.gather_qmm` over expert-sorted pairs,
bigrig_engine/stream.py:1320-1336, 1623-1626), as the layer forms here do inside their kernels; it trains
nothing. `product` is the same step for experts held in bfloat16 or float16 by the program itself,
with the gradients that tuning them, or what stands before them, takes. Rows come in the order of
`dispatch.dispatch`, with its plan's offsets; the order needs no host read, so a step can be captured.

Products run on the matrix instructions, sums are float32 and rounded once. Gradients are taken once
(create_graph=True is refused). Every result is the same bits on every run. Streams, tangents and recorders as in `dispatch`.
"""
from __future__ import annotations

import torch

from . import lib as L
from .dispatch import MAX_EXPERTS, MAX_PAIRS, MAX_WIDTH, _once, _recorded
from .mx import _handle, _on_device

MAX_ROW_STRIDE = 1 << 20    # values between a matrix's rows

_TYPES = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def _strides(w):
    """Values between experts and rows of weights [E, N, K]."""
    E, N, K = w.shape
    row = w.stride(1) if N > 1 else K
    return (w.stride(0) if E > 1 else N * row), row


def _aligned(x):
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _forward(rows, weight, offsets, bias):
    device = _on_device(rows, weight, offsets, bias)
    E, N, K = weight.shape
    out = rows.new_empty((rows.shape[0], N))
    L.check(L.load().brx_grouped_product(rows.data_ptr(), weight.data_ptr(), *_strides(weight), L.ptr(bias),
                                         offsets.data_ptr(), rows.shape[0], E, K, N, _TYPES[rows.dtype],
                                         out.data_ptr(), _handle(device)))
    return out


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, offsets, bias):
        need_rows, need_weight = ctx.needs_input_grad[:2]
        ctx.save_for_backward(rows if need_weight else None, weight if need_rows else None, offsets)
        ctx.sizes = weight.shape
        return _forward(rows, weight, offsets, bias)

    @staticmethod
    @_once
    def backward(ctx, dout):
        rows, weight, offsets = ctx.saved_tensors
        E, N, K = ctx.sizes
        dout = _aligned(dout)
        P = dout.shape[0]
        need_rows, need_weight, _, need_bias = ctx.needs_input_grad
        drows = dout.new_empty((P, K)) if need_rows else None
        dweight = dout.new_empty((E, N, K)) if need_weight else None
        dbias = dout.new_empty((E, N)) if need_bias else None
        ptr = L.ptr
        rc = L.load().brx_grouped_product_backward(
            dout.data_ptr(), ptr(rows), ptr(weight), *(_strides(weight) if need_rows else (0, K)), offsets.data_ptr(), P, E,
            K, N, _TYPES[dout.dtype], ptr(drows), ptr(dweight), ptr(dbias), _handle(dout.get_device()))
        if rc:
            L.check(rc)
        return drows, dweight, None, dbias


def product(rows, weight, offsets, bias=None, stream=None):
    """out [P, N]: row r of expert e's run, offsets[e] <= r < offsets[e + 1], is weight[e] rows[r] (+ bias[e]); the rows
    behind the last run are 0. rows [P, K] and weight [E, N, K] bfloat16 or float16 (the matrices may lie apart or be
    parts of larger ones: their rows contiguous), offsets int32 [E + 1] on the GPU, not decreasing, its first entry taken
    as 0 (`dispatch.plan`'s), bias [E, N]. K and N multiples of 8. Gradients of rows, weight and bias."""
    if stream is not None:
        return L.on_stream(stream, product, rows, weight, offsets, bias)
    if rows.dtype not in _TYPES or weight.dtype != rows.dtype or (bias is not None and bias.dtype != rows.dtype):
        raise ValueError(f"rows, weight and bias must be of one type, bfloat16 or float16, got {rows.dtype}, {weight.dtype}"
                         + ("" if bias is None else f" and {bias.dtype}"))
    if weight.dim() != 3 or rows.dim() != 2 or rows.shape[1] != weight.shape[2]:
        raise ValueError(f"rows {tuple(rows.shape)} and weight {tuple(weight.shape)} are not [P, K] and [E, N, K]")
    E, N, K = weight.shape
    P = rows.shape[0]
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"{E} experts outside [1, {MAX_EXPERTS}]")
    if P > MAX_PAIRS:
        raise ValueError(f"{P} rows in one call: at most {MAX_PAIRS}")
    for v in (K, N):
        if v % 8 or not 8 <= v <= MAX_WIDTH:
            raise ValueError(f"width {v}: a multiple of 8 up to {MAX_WIDTH}")
    if offsets.dtype != torch.int32 or offsets.shape != (E + 1,):
        raise ValueError(f"offsets must be int32 [{E + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    if bias is not None and bias.shape != (E, N):
        raise ValueError(f"bias {tuple(bias.shape)}, the weights take {(E, N)}")
    expert, row = _strides(weight)
    if weight.stride(2) != 1 or row % 8 or not K <= row <= MAX_ROW_STRIDE or expert % 8 or weight.data_ptr() % 16:
        raise ValueError(f"weight of strides {weight.stride()}: rows contiguous, 16-byte aligned, at most {MAX_ROW_STRIDE} "
                         f"values apart")
    rows = _aligned(rows)
    offsets = offsets.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if _recorded(rows, weight, bias):
        return _Product.apply(rows, weight, offsets, bias)
    return _forward(rows, weight, offsets, bias)

"""MXFP4 rows, and expert layers whose activations are MXFP4 too, on libbrx.

The reference keeps gpt-oss-style experts in MXFP4 and multiplies them by unquantized activations
(bigrig_engine/stream.py:1623-1625); so do `layer.moe_forward` and the blocks built on it. Here both
operands are MXFP4 and the products run on the scaled matrix instructions of gfx950 as the rows are
packed. That is a choice of precision, made per operator (`StreamingSwitchGLU(...,
activations="mxfp4")`): a group of 32 activations keeps e2m1's one mantissa bit under a common power
of two.

* `quantize` / `dequantize`: rows into MXFP4 and back;
* `pack_experts`: unquantized expert weights into the packed bytes of MXFP4 experts, on the GPU
  (`formats.quantize_mxfp4` of every projection, in blob layout);
* `expert_product`: one projection's rows for a list of (token, expert) pairs;
* `moe_forward` / `forward_pairs`: the layer forms of `layer.moe_forward` / `layer.forward_pairs`;
* `combine`: the weighted sum of float32 rows that `moe_forward` makes, for rows of `forward_pairs`.

A row [K] is K / 2 bytes of e2m1 codes (two a byte, the low nibble first) and K / 32 e8m0 scale
bytes, as an expert's `weight` and `scales` components hold it. A group that holds a NaN or an
infinity is held as NaN.

Tensors live on the current device. Scratch is allocated per call by torch, on the call's stream, so
calls on several streams do not share any, and a captured graph keeps its own. Given a `stream`, the
whole call runs there, its allocations and copies too; the inputs have to be ready on it (they may be freed
as soon as the call returns), and its results may be read on the stream that was current once that waits
for it.

A pool's admissions, its table and its calls wait for each other on whatever streams they are (a stream of torch's;
one made elsewhere has to outlive the pool's next admission, upload, sync or check). Replays of captured
calls are the caller's to order with them.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple

import torch

from . import formats as F
from . import lib as L
from .pool import ExpertPool
from .spec import LayerSpec

MAX_TOKENS = 65535      # token rows of one layer call
MAX_PAIRS = 1 << 21     # (token, expert) pairs of one call (a layer's shared ones too)
MAX_CODES = (1 << 32) - 257   # bytes of the codes of one call's activations
FEW_PAIRS = 64          # pairs an expert product runs without scratch


# the current device and its current stream's handle (read without building a Stream object, where this
# torch has the calls for it)
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


class MXRows(NamedTuple):
    """Rows [..., K] in MXFP4: `codes` uint8 [..., K / 2], `scales` uint8 [..., K / 32]."""
    codes: object
    scales: object

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:-1], 2 * self.codes.shape[-1])


@functools.lru_cache(maxsize=None)
def _dtype(t) -> int:
    dt = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}.get(t)
    if dt is None:
        raise ValueError(f"{t}: MXFP4 rows are made of float32, bfloat16 or float16 values")
    return dt


def _on_device(*tensors) -> int:
    """The current device; every tensor given is on it."""
    cur = -1
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d != cur or d < 0:
                if d < 0:
                    raise ValueError("tensors must be on the GPU")
                if d != _current():
                    raise ValueError(f"tensor on {t.device}, the current device is cuda:{_current()}")
                cur = d
    return cur


def _matrices(t, what: str):
    """(batch, rows, batch stride, row stride) of t [..., rows, n] seen as a run of matrices, in
    elements; its innermost dimension must be contiguous and the leading ones collapse to one."""
    n = t.dim()
    if n == 0:
        raise ValueError(f"{what} has no dimensions")
    if t.numel() == 0:
        return 0, 0, 0, 0
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what}'s innermost dimension must be contiguous (stride {t.stride(-1)})")
    if n == 2:
        return 1, t.shape[0], 0, t.stride(0)
    if n == 1:
        return 1, 1, 0, 0
    if t.is_contiguous():
        return 1, t.numel() // t.shape[-1], 0, t.shape[-1]
    if n > 3:
        try:
            t = t.view(-1, *t.shape[-2:])
        except RuntimeError:
            raise ValueError(f"{what}'s leading dimensions {tuple(t.shape[:-2])} do not collapse "
                             f"into one: make it contiguous") from None
    return t.shape[0], t.shape[1], t.stride(0), t.stride(1)


def _packed(t, what: str):
    """(batch, rows, batch stride) of packed bytes [..., rows, n] whose matrices are contiguous."""
    if t.dtype != torch.uint8:
        raise ValueError(f"{what} are uint8, got {t.dtype}")
    b, r, bs, rs = _matrices(t, what)
    if r > 1 and rs != t.shape[-1]:
        raise ValueError(f"{what}: the rows of a matrix must follow one another")
    return b, r, bs


def quantize(x, stream=None) -> MXRows:
    """x [..., K] (float32, bfloat16 or float16; K a multiple of 32; rows may be strided) in MXFP4:
    per group of 32, e = floor(log2(max |v|)) - 2 and codes v / 2^e rounded to nearest even,
    saturating at 6 -- the codes of `formats.quantize_mxfp4`. A group with a NaN or an infinity is
    held as NaN (scale byte 255)."""
    if stream is not None:
        return L.on_stream(stream, quantize, x)
    device = _on_device(x)
    dt = _dtype(x.dtype)
    shape = x.shape
    if not shape or shape[-1] % 32:
        raise ValueError(f"rows of {tuple(shape)}: the innermost dimension must be a multiple of 32")
    K = shape[-1]
    n = x.numel()
    if n and x.is_contiguous():
        b, r, bs, rs = 1, n // K, 0, K
    else:
        b, r, bs, rs = _matrices(x, "x")
    lead = shape[:-1]
    codes = x.new_empty((*lead, K // 2), dtype=torch.uint8)
    scales = x.new_empty((*lead, K // 32), dtype=torch.uint8)
    if b:
        L.check(L.load().brx_mx_quantize(x.data_ptr(), dt, b, r, K, bs, rs, codes.data_ptr(), r * (K // 2),
                                         scales.data_ptr(), r * (K // 32), _handle(device)))
    return MXRows(codes, scales)


def dequantize(q: MXRows, dtype=None, stream=None):
    """The values of q as a contiguous [..., K] tensor of `dtype` (default bfloat16; exact in
    float32 and bfloat16, rounded to nearest even in float16)."""
    if stream is not None:
        return L.on_stream(stream, dequantize, q, dtype)
    dtype = torch.bfloat16 if dtype is None else dtype
    dt = _dtype(dtype)
    codes, scales = q
    device = _on_device(codes, scales)
    shape = codes.shape
    lead = shape[:-1]
    K = 2 * shape[-1] if shape else 0
    if K % 32 or scales.shape != lead + (K // 32,):
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not "
                         f"[..., K / 2] and [..., K / 32] of one K")
    out = codes.new_empty((*lead, K), dtype=dtype)
    n = out.numel()
    if n == 0:
        return out
    if codes.is_contiguous() and scales.is_contiguous() and codes.dtype == scales.dtype == torch.uint8:
        b, r, cbs, sbs = 1, n // K, 0, 0
    else:
        b, r, cbs = _packed(codes, "codes")
        b2, r2, sbs = _packed(scales, "scales")
        if (b, r) != (b2, r2):      # one of the two is contiguous as a whole, the other is not
            if b == 1:
                b, r, cbs = b2, r2, r2 * (K // 2)
            else:
                sbs = r * (K // 32)
    L.check(L.load().brx_mx_dequantize(codes.data_ptr(), cbs, scales.data_ptr(), sbs, b, r, K, dt,
                                       out.data_ptr(), _handle(device)))
    return out


def pack_experts(spec: LayerSpec, weights: dict, biases: dict | None = None, shared: bool = False,
                 stream=None):
    """uint8 [E, bytes_per_expert]: the packed MXFP4 experts of a layer whose unquantized weights
    are weights[projection] [E, n_out, n_in] (and biases[projection] [E, n_out]), in the layout
    `ExpertPool.admit_device` and `HostStore` take. `shared`: the shared expert's width."""
    if stream is not None:
        return L.on_stream(stream, pack_experts, spec, weights, biases, shared)
    if spec.quant.mode != "mxfp4":
        raise ValueError(f"the layer's experts are {spec.quant.mode}, not mxfp4")
    es = spec.expert_spec(shared)
    if set(weights) != set(es):
        raise ValueError(f"weights for {sorted(weights)}, the layer's projections are {sorted(es)}")
    if bool(biases) != spec.has_bias or (biases and set(biases) != set(es)):
        raise ValueError(f"biases for {sorted(biases or {})}: the layer has "
                         f"{'one a projection' if spec.has_bias else 'none'}")
    E = next(iter(weights.values())).shape[0]
    for p, comps in es.items():
        n, kb = comps["scales"]["shape"]
        if tuple(weights[p].shape) != (E, n, kb * 32):
            raise ValueError(f"{p}: weights {tuple(weights[p].shape)}, the layer has {(E, n, kb * 32)}")
        if biases and tuple(biases[p].shape) != (E, n):
            raise ValueError(f"{p}: bias {tuple(biases[p].shape)}, the layer has {(E, n)}")
        _dtype(weights[p].dtype)
    device = _on_device(*weights.values(), *(biases or {}).values())
    offs, per = F.spec_offsets(es), F.spec_bytes(es)
    out = torch.empty((E, per), dtype=torch.uint8, device=next(iter(weights.values())).device)
    for p in es:
        w = weights[p]
        if w.dim() == 3 and w.is_contiguous():
            # seen as one run of rows, but every expert's codes have a place of their own
            args = (E, w.shape[1], w.shape[2], w.stride(0), w.stride(1))
        else:
            b, r, bs, rs = _matrices(w, p)
            args = (b, r, w.shape[2], bs, rs)
        if out.numel():
            L.check(L.load().brx_mx_quantize(w.data_ptr(), _dtype(w.dtype), *args,
                                             out.data_ptr() + offs[(p, "weight")], per,
                                             out.data_ptr() + offs[(p, "scales")], per, _handle(device)))
        if biases:
            o = offs[(p, "bias")]
            b16 = biases[p].to(torch.bfloat16).contiguous().view(torch.uint8)
            out[:, o:o + b16.shape[1]] = b16
    return out


# ------------------------------------------------------------------ products
def _check_spec(spec: LayerSpec) -> None:
    if spec.quant.mode != "mxfp4":
        raise ValueError(f"MXFP4 activations need MXFP4 experts, the layer's are {spec.quant.mode}")


def _check_sizes(T: int, n: int, width: int) -> None:
    """T activation rows of `width` values, n pairs: what the kernels' 32-bit counts and offsets hold."""
    if n > MAX_PAIRS:
        raise ValueError(f"{n} pairs in one call: at most {MAX_PAIRS}")
    if n and T * (width // 2) > MAX_CODES:
        raise ValueError(f"{T} rows of {width} values in one call: at most {MAX_CODES // (width // 2)}")


def _index(t, n: int, what: str):
    if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of {n} entries, got "
                         f"{t.dtype} {tuple(t.shape)}")


def _workspace(spec: LayerSpec, T: int, pairs: int, shared: bool, call: int, like):
    """Scratch for one call (L.MX_*), from torch's allocator (on the device of tensor `like`)."""
    known = spec.__dict__.setdefault("_mx_workspace", {})     # sizes, not memory
    key = (T, pairs, shared, call)
    n = known.get(key)
    if n is None:
        out = C.c_size_t()
        L.check(L.load().brx_mx_workspace_bytes(C.byref(spec.c_desc), T, pairs, int(shared),
                                                call, C.byref(out)))
        if len(known) > 4096:
            known.clear()
        n = known[key] = out.value
    return like.new_empty(n, dtype=torch.uint8)


_PROJ = {"gate_proj": 0, "up_proj": 1, "down_proj": 2}
_MLP_PROJ = {"fc1": 0, "fc2": 2}


def expert_product(spec: LayerSpec, pool: ExpertPool, q: MXRows, pair_token, pair_expert, proj: str,
                   pair_row=None, out=None, stream=None):
    """Rows W_proj[pair_expert[i]] . q[pair_token[i]] (+ bias) of one projection ("gate_proj",
    "up_proj", "down_proj"; "fc1", "fc2"), bf16 [n_pairs, n_out]. q: the activations [T, n_in];
    pair_token and pair_expert int32 [n_pairs] (entries outside are clamped, as in the layer's pair
    lists). With `out` [n_rows, n_out] and pair_row (distinct rows), row pair_row[i] is written and
    the others are left as they are. Up to 64 pairs run as one launch and without scratch, more
    as one or two; the rows are the same bits."""
    if stream is not None:
        return L.on_stream(stream, expert_product, spec, pool, q, pair_token, pair_expert, proj, pair_row, out)
    _check_spec(spec)
    j = (_PROJ if spec.gated else _MLP_PROJ).get(proj)
    if j is None:
        raise ValueError(f"projection {proj!r} not in {list(_PROJ if spec.gated else _MLP_PROJ)}")
    n_out, n_in = (spec.hidden, spec.inter) if j == 2 else (spec.inter, spec.hidden)
    codes, scales = q
    n = pair_expert.numel()
    T = codes.shape[0] if codes.dim() else 0
    _check_sizes(T, n, n_in)
    device = _on_device(codes, scales, pair_token, pair_expert, pair_row, out)
    if codes.shape != (T, n_in // 2) or scales.shape != (T, n_in // 32):
        raise ValueError(f"activations {tuple(codes.shape)} / {tuple(scales.shape)}: {proj} takes rows "
                         f"of {n_in} values")
    if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not codes.is_contiguous() or
            not scales.is_contiguous()):
        raise ValueError("activations must be contiguous uint8 codes and scales")
    _index(pair_token, n, "pair_token")
    _index(pair_expert, n, "pair_expert")
    if pair_row is not None:
        _index(pair_row, n, "pair_row")
        if out is None:
            raise ValueError("pair_row names rows of an `out` that is not given")
    if out is None:
        out = codes.new_empty((n, n_out), dtype=torch.bfloat16)
    elif out.dtype != torch.bfloat16 or out.dim() != 2 or out.shape[1] != n_out or not out.is_contiguous():
        raise ValueError(f"out must be contiguous bfloat16 [n_rows, {n_out}]")
    ws = _workspace(spec, T, n, False, L.MX_PRODUCT, codes) if n > FEW_PAIRS else None
    L.check(L.load().brx_mx_expert_product(
        C.byref(spec.c_desc), pool.device.handle, codes.data_ptr(), scales.data_ptr(), T, pair_token.data_ptr(),
        pair_expert.data_ptr(), None if pair_row is None else pair_row.data_ptr(), n, out.shape[0], j,
        out.data_ptr(), None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), _handle(device)))
    return out


def _rows_of(spec: LayerSpec, x):
    if x.dtype != torch.bfloat16 or not x.shape or x.shape[-1] != spec.hidden:
        raise ValueError(f"x must be bfloat16 [..., {spec.hidden}], got {x.dtype} {tuple(x.shape)}")
    return x if x.dim() == 2 and x.is_contiguous() else x.reshape(-1, spec.hidden).contiguous()


def moe_forward(spec: LayerSpec, pool: ExpertPool, x, idx, w=None, shared=None, sgate=None, out=None,
                y_unreduced=None, flags=None, stream=None):
    """The routed experts of tokens x [T, H] (bf16) under a routing idx [T, k] (int32) with both
    projections' activations in MXFP4. With weights w [T, k] (fp32): out [T, H] = sum_j w[t, j] *
    y[t, j] (+ sgate[t] * shared(x_t)) over the float32 rows y; without: the unreduced rows [T, k, H] in
    bfloat16. The pool's table must
    be uploaded (`ExpertPool.g2s_device`), as for `layer.moe_forward`. Few pairs run
    as two or three launches, the rest as the grouped GEMM; the outputs are the same bits (`flags`:
    BRX_FWD_FORCE_DECODE for the first, up to 8 tokens and 64 pairs, BRX_FWD_FORCE_PREFILL for the last)."""
    if stream is not None:
        return L.on_stream(stream, moe_forward, spec, pool, x, idx, w, shared, sgate, out, y_unreduced, flags)
    _check_spec(spec)
    x2 = _rows_of(spec, x)
    T, H, k = x2.shape[0], spec.hidden, spec.top_k
    if T > MAX_TOKENS:
        raise ValueError(f"{T} tokens in one call: at most {MAX_TOKENS}")
    _check_sizes(T, T * k, H)
    device = _on_device(x2, idx, w, shared, sgate, out, y_unreduced)
    _index(idx, T * k, "idx")
    if w is not None and (w.dtype != torch.float32 or w.numel() != T * k or not w.is_contiguous()):
        raise ValueError(f"w must be contiguous float32 [{T}, {k}]")
    if sgate is not None and (sgate.dtype != torch.float32 or sgate.numel() != T or not sgate.is_contiguous()):
        raise ValueError(f"sgate must be contiguous float32 [{T}]")
    if shared is not None:
        _check_shared(spec, shared)
    for t, n in ((out, T * H), (y_unreduced, T * k * H)):
        if t is not None and (t.dtype != torch.bfloat16 or t.numel() != n or not t.is_contiguous()):
            raise ValueError(f"out and y_unreduced must be contiguous bfloat16 [{T}, {H}] and [{T}, {k}, {H}]")
    if w is not None and out is None:
        out = x2.new_empty((T, H))
    if w is None and y_unreduced is None:
        y_unreduced = x2.new_empty((T, k, H))
    ws = _workspace(spec, T, T * k, shared is not None, L.MX_ROWS if out is None else L.MX_LAYER, x2)
    ptr = L.ptr
    L.check(L.load().brx_mx_moe_forward(
        C.byref(spec.c_desc), pool.device.handle, x2.data_ptr(), idx.data_ptr(), ptr(w), ptr(shared),
        ptr(sgate), T, ptr(out), ptr(y_unreduced), 0 if flags is None else flags, ws.data_ptr(), ws.numel(),
        _handle(device)))
    return out if w is not None else y_unreduced


def _check_shared(spec: LayerSpec, shared) -> None:
    if not spec.shared_inter:
        raise ValueError("the layer has no shared expert")
    per = spec.__dict__.get("_mx_shared_bytes")
    if per is None:
        per = spec.__dict__["_mx_shared_bytes"] = F.spec_bytes(spec.expert_spec(True))
    if shared.dtype != torch.uint8 or shared.numel() != per or not shared.is_contiguous():
        raise ValueError(f"the shared expert is {per} contiguous bytes")


def forward_pairs(spec: LayerSpec, pool: ExpertPool, x, pair_tok, pair_exp, pair_row, y_rows, flags: int,
                  shared=None, stream=None) -> None:
    """`layer.forward_pairs` with MXFP4 activations (any `flags` give the same bits); y_rows bfloat16, or
    float32 for `combine`."""
    if stream is not None:
        return L.on_stream(stream, forward_pairs, spec, pool, x, pair_tok, pair_exp, pair_row, y_rows, flags, shared)
    _check_spec(spec)
    x2 = _rows_of(spec, x)
    n = pair_exp.numel()
    _check_sizes(x2.shape[0], n, spec.hidden)
    device = _on_device(x2, pair_tok, pair_exp, pair_row, y_rows, shared)
    _index(pair_tok, n, "pair_tok")
    _index(pair_exp, n, "pair_exp")
    if pair_row is not None:
        _index(pair_row, n, "pair_row")
    if shared is not None:
        _check_shared(spec, shared)
    if (y_rows.dtype not in (torch.bfloat16, torch.float32) or y_rows.dim() != 2 or
            y_rows.shape[1] != spec.hidden or not y_rows.is_contiguous()):
        raise ValueError(f"y_rows must be contiguous bfloat16 or float32 [n_rows, {spec.hidden}]")
    ws = _workspace(spec, x2.shape[0], n, shared is not None, L.MX_ROWS, x2)
    ptr = L.ptr
    L.check(L.load().brx_mx_moe_forward_pairs(
        C.byref(spec.c_desc), pool.device.handle, x2.data_ptr(), x2.shape[0], ptr(pair_tok), ptr(pair_exp),
        ptr(pair_row), n, y_rows.shape[0], ptr(shared), y_rows.data_ptr(), _dtype(y_rows.dtype), flags, ws.data_ptr(), ws.numel(),
        _handle(device)))


def combine(spec: LayerSpec, y_routed, w, out, y_shared=None, sgate=None, stream=None) -> None:
    """out[t] = sum_j w[t, j] * y_routed[t, j] (+ sgate[t] * y_shared[t]): rows float32 [T k, H] and
    [T, H], w and sgate float32, out bfloat16 [T, H]."""
    if stream is not None:
        return L.on_stream(stream, combine, spec, y_routed, w, out, y_shared, sgate)
    T, H, k = out.shape[0], spec.hidden, spec.top_k
    device = _on_device(out, y_routed, w, y_shared, sgate)
    if out.dtype != torch.bfloat16 or out.shape != (T, H) or not out.is_contiguous():
        raise ValueError(f"out must be contiguous bfloat16 [T, {H}]")
    for t, n, what in ((y_routed, T * k * H, "y_routed"), (w, T * k, "w"), (y_shared, T * H, "y_shared"), (sgate, T, "sgate")):
        if t is not None and (t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous()):
            raise ValueError(f"{what} must be {n} contiguous float32 values")
    ptr = L.ptr
    L.check(L.load().brx_mx_combine(C.byref(spec.c_desc), ptr(y_routed), ptr(w), ptr(y_shared), ptr(sgate), T,
                                    out.data_ptr(), _handle(device)))

"""MXFP4 in 64 bits, from the definition: rounding rows, the values of codes, products and the expert
layer with MXFP4 activations, each with a bound of what the kernels' fp32 arithmetic may be off by.

The bounds. A product's terms are exact (a 4-bit by 4-bit significand times a power of two), so a
sum of K terms in fp32, whatever its order, is off by at most about one rounding an addition that
the partial sums go through, relative to the sum of the terms' magnitudes: `SUM(K)` counts one per
128-term step and 8 for the adds inside a step, and for a kernel that adds partial sums of its own,
at 2^-23 each (twice a rounding to nearest, for hardware that truncates). The activation is off by
its inputs' errors times its derivatives plus 16 roundings of its own (hardware exp2 and reciprocal,
1 ulp each, among them; exp2 of an argument of up to ~2^7 carries 2^-24 * 2^7 relative).
A rounding to bf16 is off by at most 2^-8 of the value."""
import numpy as np

from bigrig_amd import formats as F

MAGS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def SUM(K):
    return (-(-K // 128) + 8) * 2.0 ** -23


def scale_of(a):
    """The group exponent of largest magnitude a (float64 array)."""
    m, ex = np.frexp(a)
    return np.clip(np.where(a > 0, ex - 3, -127), -127, 127)


def to_codes(v):
    """e2m1 codes of v (already divided by the scale): nearest, ties to the even code, saturating."""
    a = np.minimum(np.abs(v), 6.0)
    hi = np.searchsorted(MAGS, a)                 # the first magnitude not below a
    lo = np.maximum(hi - 1, 0)
    up = (MAGS[hi] - a < a - MAGS[lo]) | ((MAGS[hi] - a == a - MAGS[lo]) & (hi % 2 == 0))
    c = np.where(up, hi, lo)
    return np.where((v < 0) & (c > 0), c + 8, c).astype(np.uint8)


def quantize(x):
    """(codes [..., K] one a value, scale bytes [..., K / 32]) of float64 x [..., K]."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    a = np.abs(g).max(-1)
    bad = ~np.isfinite(a)
    e = scale_of(np.where(bad, 0, a))
    with np.errstate(invalid="ignore"):
        c = to_codes(np.where(bad[..., None], 0, g) / np.exp2(e.astype(np.float64))[..., None])
    return (np.where(bad[..., None], 0, c).astype(np.uint8).reshape(x.shape),
            np.where(bad, 255, e + 127).astype(np.uint8))


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def values(codes, scales):
    """float64 values of one-a-value codes."""
    v = np.where(codes >= 8, -1.0, 1.0) * MAGS[codes & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*codes.shape[:-1], -1, 32) * s[..., None]).reshape(codes.shape)


def held(x):
    return values(*quantize(x))


def weights(spec, blob, proj, shared=False):
    """(float64 weights [n_out, n_in], bias [n_out]) of a packed expert."""
    arr = F.split_expert(blob, spec.expert_spec(shared))
    w = F.dequantize_projection(arr, proj, spec.quant).astype(np.float64)
    b = arr.get((proj, "bias"))
    return w, np.zeros(w.shape[0]) if b is None else F.bf16_bits_to_f32(b).astype(np.float64)


def product(w, b, x):
    """(x W^T + b, its bound in fp32) of held rows x."""
    return x @ w.T + b, SUM(x.shape[1]) * (np.abs(x) @ np.abs(w).T + np.abs(b))


def activation(spec, g, dg, u, du):
    """(act(g, u), bound) for inputs off by at most dg, du."""
    def silu(v, a):
        s = 1.0 / (1.0 + np.exp(-a * v))
        return v * s, s * (1.0 + np.abs(a * v) * (1.0 - s))      # value, bound of the slope
    if spec.act == "silu_mlp":
        h, d = silu(g, 1.0)
        return h, d * dg + (16 + 2 * np.abs(g)) * 2.0 ** -23 * np.abs(h)
    if spec.act == "swiglu_clamped":
        gc, uc = np.minimum(g, spec.limit), np.clip(u, -spec.limit, spec.limit) + 1.0
        s, d = silu(gc, spec.alpha)
    else:
        gc, uc = g, u
        s, d = silu(g, 1.0)
    h = s * uc
    return h, np.abs(uc) * d * dg + np.abs(s) * (du + 2.0 ** -23 * np.abs(uc)) + (16 + 4 * np.abs(gc)) * 2.0 ** -23 * np.abs(h)


def held_bounded(h, dh):
    """(held(h), how far the held value of anything within dh of h may be from it): the group's
    exponent and the element's code may each fall either way of a border that dh reaches."""
    q = held(h)
    g, d = h.reshape(*h.shape[:-1], -1, 32), dh.reshape(*h.shape[:-1], -1, 32)
    lo = scale_of(np.maximum(np.abs(g) - d, 0).max(-1))
    hi = scale_of((np.abs(g) + d).max(-1))
    far = np.zeros(g.shape)
    for e in (lo, hi):
        s = np.exp2(e.astype(np.float64))[..., None]
        for v in (g - d, g + d):
            c = to_codes(v / s)
            r = np.where(c >= 8, -1.0, 1.0) * MAGS[c & 7] * s
            far = np.maximum(far, np.abs(r - q.reshape(g.shape)))
    return q, far.reshape(h.shape)


def expert_rows(spec, blob, xq, shared=False):
    """(fp64 rows y, bound before any rounding of y) of one expert for held rows xq."""
    es = list(spec.expert_spec(shared))
    w, b = weights(spec, blob, es[0], shared)
    g, dg = product(w, b, xq)
    u = du = 0.0
    if len(es) == 3:
        w, b = weights(spec, blob, es[1], shared)
        u, du = product(w, b, xq)
    h, dh = activation(spec, g, dg, u, du)
    q, far = held_bounded(h, dh)
    w, b = weights(spec, blob, es[-1], shared)
    y, dy = product(w, b, q)
    return y, dy + far @ np.abs(w).T * (1 + SUM(q.shape[1]))


def layer(spec, experts, x, idx, w=None, shared=None, sgate=None):
    """(y [T, k, H], bound, out [T, H] or None, bound): x float64 [T, H]. y is rounded to bf16, out is the
    sum of the rows as they were before, rounded once."""
    T, k = idx.shape
    xq = held(x)
    y, dy = np.zeros((T, k, spec.hidden)), np.zeros((T, k, spec.hidden))
    for e in np.unique(idx):
        t, j = np.nonzero(idx == e)
        y[t, j], dy[t, j] = expert_rows(spec, experts[e], xq[t])
    dy16 = dy + 2.0 ** -8 * (np.abs(y) + dy)
    if w is None:
        return y, dy16, None, None
    w = w.astype(np.float64)
    out = (w[..., None] * y).sum(1)
    dout = (np.abs(w)[..., None] * dy).sum(1)
    mag = (np.abs(w)[..., None] * np.abs(y)).sum(1)
    if shared is not None:
        s, ds = expert_rows(spec, shared, xq, True)
        sg = sgate.astype(np.float64)[:, None]
        out, mag = out + sg * s, mag + np.abs(sg * s)
        dout = dout + np.abs(sg) * ds
    dout = dout + (k + 2) * 2.0 ** -23 * mag
    return y, dy16, out, dout + 2.0 ** -8 * (np.abs(out) + dout)

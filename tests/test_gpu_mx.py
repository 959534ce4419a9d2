"""MXFP4 rows, expert products and the layer with MXFP4 activations on the GPU, against the 64-bit
restatement in mx_oracle (codes and scales equal; products and layers within its bounds)."""
import ctypes as C

import numpy as np
import pytest

from bigrig_amd import formats as F
from bigrig_amd import lib as L
from bigrig_amd import mx
from bigrig_amd.layer import MoELayer, StreamingSwitchGLU
from bigrig_amd.layer import moe_forward as _bf16_forward
from bigrig_amd.pool import ExpertPool, HostStore, PinnedFetcher
from bigrig_amd.spec import E256_SHARED, GPT_OSS_120B, OLMOE_1B_7B, QWEN3_30B_A3B
from tests import mx_oracle as O
from tests.gpu_util import bits, build_gpu_layer, bytes_dev, to_dev_bits
from tests.helpers import make_layer, small

pytestmark = pytest.mark.gpu

MX = F.QuantSpec(4, 32, "mxfp4")
# widths that end inside a 128-K step (64 more) and inside the blocks' 32-, 64-, 128- and 256-row runs
SWIGLU = small(QWEN3_30B_A3B, quant=MX, hidden=320, inter=192, n_experts=6, top_k=2)
SHARED = small(E256_SHARED, quant=MX, hidden=256, inter=64, shared_inter=448, n_experts=8, top_k=3)
CLAMPED = small(GPT_OSS_120B, hidden=192, inter=576, n_experts=5, top_k=4)
MLP = small(OLMOE_1B_7B, quant=MX, hidden=64, inter=320, n_experts=4, top_k=1, act="silu_mlp", has_bias=True)
WIDE = small(GPT_OSS_120B, hidden=2880, inter=64, n_experts=3, top_k=2)
LONG = small(QWEN3_30B_A3B, quant=MX, hidden=64, inter=8192, n_experts=2, top_k=1)
SPECS = {"swiglu": SWIGLU, "shared": SHARED, "clamped": CLAMPED, "mlp": MLP, "wide": WIDE, "long": LONG}


def acts(T, H, seed, big=20.0):
    """bf16 bit patterns [T, H]: N(0, 1) with a few large channels."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, H), dtype=np.float32)
    x[:, rng.integers(0, H, max(1, H // 64))] *= big
    return F.f32_to_bf16_bits(x)


def f64(b):
    return F.bf16_bits_to_f32(b).astype(np.float64)


def routing(spec, T, seed):
    rng = np.random.default_rng(seed)
    p = 1.0 / (np.arange(spec.n_experts) + 1.0)
    idx = np.stack([rng.choice(spec.n_experts, spec.top_k, replace=False, p=p / p.sum()) for _ in range(T)])
    w = rng.random((T, spec.top_k), dtype=np.float32) + 0.1
    return idx.astype(np.int32), (w / w.sum(1, keepdims=True)).astype(np.float32)


def dev(a, gpu):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


_LAYERS = {}


def built(name, gpu):
    """(spec, oracle layer, switch with MXFP4 activations, pool) of SPECS[name], every expert resident."""
    import torch
    if name not in _LAYERS:
        lay = make_layer(SPECS[name], seed=600 + sorted(SPECS).index(name), expert_std=0.05)
        _, sw, pool, _ = build_gpu_layer(lay, gpu)
        sw.activations = "mxfp4"
        pool.g2s_device(torch.cuda.current_stream().cuda_stream)
        _LAYERS[name] = (lay.spec, lay, sw, pool)
    return _LAYERS[name]


def layer_forward(spec, pool, x, idx, w):
    """The layer with bf16 activations."""
    import torch
    out = torch.empty((x.shape[0], spec.hidden), dtype=torch.bfloat16, device=x.device)
    _bf16_forward(spec, pool, x, idx, w, out=out)
    return out


def close(got, want, bound, what):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside, worst "
                           f"{np.max(np.abs(got - want) / np.maximum(bound, 1e-300)):.3g} of the bound")


# ------------------------------------------------------------------ rows
def _values(kind, rows, cols, seed):
    """float32 values that the type holds exactly."""
    rng = np.random.default_rng(seed)
    v = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 4, (rows, 1)))).astype(np.float32)
    if kind == "f16":
        return v.astype(np.float16).astype(np.float32)
    return v if kind == "f32" else F.round_bf16(v)


def _tensor(v, kind, gpu):
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]
    return torch.from_numpy(v).to(gpu).to(dt)


def _check_rows(q, v64):
    codes, scales = O.quantize(v64)
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), O.pack(codes))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (17, 96), (5, 2880), (257, 128), (1000, 416)])
def test_quantize_and_back(gpu, kind, shape):
    import torch
    v = _values(kind, *shape, seed=shape[0])
    q = mx.quantize(_tensor(v, kind, gpu))
    _check_rows(q, v.astype(np.float64))
    want = O.held(v.astype(np.float64))
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        got = mx.dequantize(q, dt)
        assert got.dtype == dt and tuple(got.shape) == shape
        exact = torch.from_numpy(want).to(dt).double().numpy()      # (a rounding in float16 only)
        assert np.array_equal(got.double().cpu().numpy(), exact)


def test_every_border_of_a_code(gpu):
    """Each value just below, at and just above every border between two codes, at several scales, the
    smallest and the largest among them."""
    cuts = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    v = np.concatenate([np.nextafter(cuts, np.float32(0)), cuts, np.nextafter(cuts, np.float32(9)),
                        np.float32([6.0, 7.0, 7.999])])
    g = np.zeros((2, 32), dtype=np.float32)
    g[0, :24], g[0, 24], g[1, :24], g[1, 24] = v, 6.0, -v, 4.0
    rows = np.concatenate([np.ldexp(g, e) for e in (-126, -60, -3, 0, 5, 100, 125)]).astype(np.float32)
    q = mx.quantize(_tensor(rows, "f32", gpu))
    _check_rows(q, rows.astype(np.float64))
    assert np.array_equal(mx.dequantize(q, __import__("torch").float32).cpu().numpy(),
                          O.held(rows.astype(np.float64)).astype(np.float32))


def test_zeros_subnormals_and_the_largest(gpu):
    import torch
    v = np.zeros((8, 32), dtype=np.float32)
    v[1] = -0.0
    v[2, 5] = np.float32(2.0 ** -149)
    v[3, 5] = np.float32(2.0 ** -127)
    v[4, 5], v[4, 6] = np.float32(1.5 * 2.0 ** -126), np.float32(-2.0 ** -128)
    v[5, 5] = np.finfo(np.float32).max
    v[6, 5], v[6, 6] = np.float32(2.0 ** 127), np.float32(1.0)
    v[7] = np.nextafter(np.float32(4.0), np.float32(0))      # just below a power of two
    q = mx.quantize(_tensor(v, "f32", gpu))
    _check_rows(q, v.astype(np.float64))
    for dt in (torch.float32, torch.bfloat16):               # (their subnormals among them)
        assert np.array_equal(mx.dequantize(q, dt).double().cpu().numpy(), O.held(v.astype(np.float64)))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_infinities_and_nan_make_their_group_nan(gpu, kind):
    import torch
    v = _values(kind, 6, 96, seed=4)
    v[0, 3], v[1, 40], v[2, 95] = np.inf, -np.inf, np.nan
    q = mx.quantize(_tensor(v, kind, gpu))
    _check_rows(q, v.astype(np.float64))
    got = mx.dequantize(q, torch.bfloat16).float().cpu().numpy()
    bad = np.zeros((6, 3), bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert np.array_equal(np.isnan(got).reshape(6, 3, 32).all(-1), bad)
    assert np.array_equal(np.isnan(got).reshape(6, 3, 32).any(-1), bad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strided_and_misaligned_rows(gpu, kind):
    import torch
    v = _values(kind, 4 * 9, 160, seed=9).reshape(4, 9, 160)
    t = _tensor(v, kind, gpu)
    for cut in (np.s_[:, ::2, :], np.s_[:, 1:4, 32:96], np.s_[1, :, 1:33], np.s_[::2, 3, 5:133], np.s_[2, 3, 7:71],
                np.s_[:, :, 3:131]):
        _check_rows(mx.quantize(t[cut]), v[cut].astype(np.float64))
    flat = t.reshape(-1)[1:1 + 32 * 40].view(40, 32)
    _check_rows(mx.quantize(flat), v.reshape(-1)[1:1 + 32 * 40].reshape(40, 32).astype(np.float64))
    one = t[0, :1].expand(5, 160)
    _check_rows(mx.quantize(one), np.repeat(v[0, :1], 5, 0).astype(np.float64))
    for shape in ((0, 32), (5, 0), (2, 0, 64)):
        q = mx.quantize(torch.zeros(shape, device=gpu))
        assert tuple(mx.dequantize(q).shape) == shape and q.shape == shape
    with pytest.raises(ValueError, match="innermost"):
        mx.quantize(t[0, :, ::2][:, :64])
    with pytest.raises(ValueError, match="multiple of 32"):
        mx.quantize(t[:, :, :33])
    with pytest.raises(ValueError, match="float64"):
        mx.quantize(t.double())


def test_offsets_past_32_bits(gpu):
    """4.6 G values (one row again and again, by a row stride of zero): every row is the first one's."""
    import torch
    row = to_dev_bits(acts(1, 65536, 12), gpu)
    q = mx.quantize(row.expand(70000, 65536))
    one = mx.quantize(row)
    assert torch.equal(q.codes[0], one.codes[0]) and torch.equal(q.scales[0], one.scales[0])
    for at in range(0, 70000, 10000):
        assert bool((q.codes[at:at + 10000] == one.codes).all()) and bool((q.scales[at:at + 10000] == one.scales).all())
    back, want = mx.dequantize(q), mx.dequantize(one)
    for at in range(0, 70000, 10000):
        assert bool((back[at:at + 10000] == want).all())


@pytest.mark.parametrize("name", ["clamped", "mlp", "swiglu", "shared"])
def test_pack_experts(gpu, name):
    import torch
    spec = SPECS[name]
    rng = np.random.default_rng(12)
    for shared in ([False, True] if spec.shared_inter else [False]):
        E = 1 if shared else 3
        es = spec.expert_spec(shared)
        w, b, blobs = {}, {}, [{} for _ in range(E)]
        for p, comps in es.items():
            n, k = comps["scales"]["shape"]
            m = F.round_bf16(rng.standard_normal((E, n, 32 * k)).astype(np.float32) * 0.05)
            w[p] = torch.from_numpy(m).to(gpu).to(torch.bfloat16)
            for e in range(E):
                blobs[e][(p, "weight")], blobs[e][(p, "scales")] = F.quantize_mxfp4(m[e])
            if spec.has_bias:
                v = F.f32_to_bf16_bits(rng.standard_normal((E, n)).astype(np.float32))
                b[p] = to_dev_bits(v, gpu)
                for e in range(E):
                    blobs[e][(p, "bias")] = v[e]
        got = mx.pack_experts(spec, w, b or None, shared).cpu().numpy()
        for e in range(E):
            assert got[e].tobytes() == F.join_expert(blobs[e], es)
        # the same weights as views of wider matrices
        wide = {p: torch.cat([t, t], 2)[:, :, :t.shape[2]] for p, t in w.items()}
        assert np.array_equal(mx.pack_experts(spec, wide, b or None, shared).cpu().numpy(), got)


def test_dequantize_reads_packed_experts(gpu):
    """A projection's components inside packed experts are matrices a batch stride apart."""
    import torch
    spec, lay, _, _ = built("clamped", gpu)
    blob = torch.stack([bytes_dev(b, gpu) for b in lay.experts])
    offs = F.spec_offsets(spec.expert_spec())
    for p, comps in spec.expert_spec().items():
        n, g = comps["scales"]["shape"]
        o, s = offs[(p, "weight")], offs[(p, "scales")]
        q = mx.MXRows(blob[:, o:o + n * g * 16].unflatten(1, (n, g * 16)), blob[:, s:s + n * g].unflatten(1, (n, g)))
        got = mx.dequantize(q, torch.float32).cpu().numpy()
        for e in range(spec.n_experts):
            assert np.array_equal(got[e].astype(np.float64), O.weights(spec, lay.experts[e], p)[0])


# ------------------------------------------------------------------ products
def _product(gpu, name, proj, T, P, seed, experts=None):
    spec, lay, _, pool = built(name, gpu)
    rng = np.random.default_rng(seed)
    k_in = spec.expert_spec()[proj]["scales"]["shape"][1] * 32
    x = acts(T, k_in, seed)
    q = mx.quantize(to_dev_bits(x, gpu))
    tok = rng.integers(0, T, P).astype(np.int32)
    ex = (rng.integers(0, spec.n_experts, P) if experts is None else np.resize(experts, P)).astype(np.int32)
    xq = O.held(f64(x))
    w = [O.weights(spec, b, proj) for b in lay.experts]
    want = np.zeros((P, w[0][0].shape[0]))
    bound = np.zeros_like(want)
    for e in range(spec.n_experts):
        i = np.flatnonzero(ex == e)
        if i.size:
            want[i], bound[i] = O.product(*w[e], xq[tok[i]])
    bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    return spec, pool, q, tok, ex, want, bound


@pytest.mark.parametrize("name, proj", [("swiglu", "gate_proj"), ("swiglu", "down_proj"), ("clamped", "up_proj"),
                                        ("clamped", "down_proj"), ("mlp", "fc1"), ("mlp", "fc2"),
                                        ("wide", "gate_proj"), ("long", "down_proj")])
@pytest.mark.parametrize("T, P", [(1, 1), (3, 16), (7, 65), (40, 333)])
def test_expert_product(gpu, name, proj, T, P):
    spec, pool, q, tok, ex, want, bound = _product(gpu, name, proj, T, P, seed=T + P)
    got = mx.expert_product(spec, pool, q, dev(tok, gpu), dev(ex, gpu), proj)
    close(f64(bits(got)), want, bound, f"{name} {proj} T={T} P={P}")


@pytest.mark.parametrize("P", [15, 17, 33, 64, 128, 200])
def test_expert_product_of_one_expert(gpu, P):
    """Every pair at one expert (one run of tiles, the last partly filled; the other experts have none)."""
    spec, pool, q, tok, ex, want, bound = _product(gpu, "swiglu", "up_proj", 9, P, seed=P, experts=[4])
    got = mx.expert_product(spec, pool, q, dev(tok, gpu), dev(ex, gpu), "up_proj")
    close(f64(bits(got)), want, bound, f"one expert P={P}")


COUNTS = [64, 80, 81, 65, 145, 144]      # a tile of 64; 16 and 17 pairs past one; 1 past; 16 and 17 past two


def test_expert_product_of_tall_tiles(gpu):
    """Pairs a little past whole tiles, which the last tile takes or does not."""
    ex = np.random.default_rng(3).permutation(np.repeat(np.arange(6), COUNTS))
    for proj in ("gate_proj", "down_proj"):
        spec, pool, q, tok, ex, want, bound = _product(gpu, "swiglu", proj, 70, len(ex), seed=8, experts=ex)
        got = mx.expert_product(spec, pool, q, dev(tok, gpu), dev(ex, gpu), proj)
        close(f64(bits(got)), want, bound, f"tall tiles {proj}")


def test_layer_of_tall_tiles(gpu):
    """The pairs form over the same counts: the rows a call of one pair each gives, bit for bit."""
    import torch
    spec, lay, sw, pool = built("swiglu", gpu)
    x = to_dev_bits(acts(8, spec.hidden, 31), gpu)
    rng = np.random.default_rng(4)
    ex = rng.permutation(np.repeat(np.arange(6), COUNTS)).astype(np.int32)
    tok = rng.integers(0, 8, ex.size).astype(np.int32)
    y = torch.zeros(ex.size, spec.hidden, dtype=torch.bfloat16, device=gpu)
    mx.forward_pairs(spec, pool, x, dev(tok, gpu), dev(ex, gpu), None, y, 0)
    each = torch.zeros(48, spec.hidden, dtype=torch.bfloat16, device=gpu)
    t48, e48 = np.repeat(np.arange(8), 6).astype(np.int32), np.tile(np.arange(6), 8).astype(np.int32)
    mx.forward_pairs(spec, pool, x, dev(t48, gpu), dev(e48, gpu), None, each, L.FWD_FORCE_DECODE)
    assert np.array_equal(bits(y), bits(each)[tok * 6 + ex])


def test_expert_product_rows(gpu):
    """pair_row scatters the rows; rows no pair names are left as they were."""
    import torch
    spec, pool, q, tok, ex, want, bound = _product(gpu, "clamped", "gate_proj", 6, 50, seed=2)
    row = np.random.default_rng(5).permutation(80)[:50].astype(np.int32)
    out = torch.full((80, want.shape[1]), 7.0, dtype=torch.bfloat16, device=gpu)
    got = mx.expert_product(spec, pool, q, dev(tok, gpu), dev(ex, gpu), "gate_proj", dev(row, gpu), out)
    assert got.data_ptr() == out.data_ptr()
    o = f64(bits(out))
    close(o[row], want, bound, "scattered rows")
    assert (o[np.setdiff1d(np.arange(80), row)] == 7.0).all()
    alone = mx.expert_product(spec, pool, q, dev(tok, gpu), dev(ex, gpu), "gate_proj")
    assert np.array_equal(bits(alone), bits(out)[row])


def test_product_refusals(gpu):
    import torch
    spec, pool, q, tok, ex, _, _ = _product(gpu, "swiglu", "gate_proj", 3, 8, seed=1)
    t, e = dev(tok, gpu), dev(ex, gpu)
    call = lambda **kw: mx.expert_product(**dict(dict(   # noqa: E731
        spec=spec, pool=pool, q=q, pair_token=t, pair_expert=e, proj="gate_proj"), **kw))
    for kw, what in ((dict(pair_token=t[:7]), "pair_token"), (dict(pair_expert=e.long()), "pair_expert"),
                     (dict(pair_row=t), "out"), (dict(proj="down_proj"), "activations"),
                     (dict(q=mx.MXRows(q.codes[:, ::2], q.scales)), "activations"),
                     (dict(q=mx.MXRows(q.codes.t().contiguous().t(), q.scales)), "contiguous"),
                     (dict(out=torch.zeros(8, 192, device=gpu)), "bfloat16"),
                     (dict(pair_token=t.cpu()), "on the GPU")):
        with pytest.raises(ValueError, match=what):
            call(**kw)
    with pytest.raises(L.BrxError, match="y_rows has 7 rows"):
        call(out=torch.zeros(7, 192, dtype=torch.bfloat16, device=gpu))
    assert tuple(call(pair_token=t[:0], pair_expert=e[:0]).shape) == (0, 192)
    d = spec.desc()
    lib = L.load()
    y = torch.zeros(8, 192, dtype=torch.bfloat16, device=gpu)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)

    def raw(codes=q.codes.data_ptr(), T=3, n=8, proj=0, w=ws.data_ptr(), nb=ws.numel(), out=y.data_ptr()):
        return lib.brx_mx_expert_product(C.byref(d), pool.device.handle, codes, q.scales.data_ptr(), T, t.data_ptr(),
                                         e.data_ptr(), None, n, 8, proj, out, w, nb, None)
    for kw in (dict(codes=None), dict(codes=q.codes.data_ptr() + 8), dict(T=0), dict(T=-1), dict(n=-1), dict(proj=3),
               dict(out=None), dict(out=y.data_ptr() + 2)):
        assert raw(**kw) == L.BRX_EINVAL, kw
    assert raw() == 0
    # more pairs take scratch
    t, e = t.repeat(10), e.repeat(10)
    y = torch.zeros(80, 192, dtype=torch.bfloat16, device=gpu)
    more = lambda w, nb: lib.brx_mx_expert_product(   # noqa: E731
        C.byref(d), pool.device.handle, q.codes.data_ptr(), q.scales.data_ptr(), 3, t.data_ptr(), e.data_ptr(), None,
        80, 80, 0, y.data_ptr(), w, nb, None)
    for w, nb in ((None, ws.numel()), (ws.data_ptr() + 16, ws.numel() - 256), (ws.data_ptr(), 64)):
        assert more(w, nb) == L.BRX_EINVAL
    assert more(ws.data_ptr(), ws.numel()) == 0
    torch.cuda.synchronize()


# ------------------------------------------------------------------ the layer
def _layer_inputs(spec, lay, gpu, T, seed):
    x = acts(T, spec.hidden, seed)
    idx, w = routing(spec, T, seed)
    sg = None
    if lay.shared is not None:
        sg = np.random.default_rng(seed).random(T, dtype=np.float32)
    return x, idx, w, sg


@pytest.mark.parametrize("name", ["swiglu", "shared", "clamped", "mlp", "wide"])
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 33, 150])
def test_layer(gpu, name, T):
    spec, lay, sw, pool = built(name, gpu)
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=T)
    out = mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), shared=sw.shared,
                         sgate=None if sg is None else dev(sg, gpu))
    rows = mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu))
    y, dy, want, bound = O.layer(spec, lay.experts, f64(x), idx, w, lay.shared, sg)
    close(f64(bits(rows)), y, dy, f"{name} rows T={T}")
    close(f64(bits(out)), want, bound, f"{name} T={T}")


def test_layer_long_width(gpu):
    """The widest intermediate: A rows of 4 KB, tiles of fewer pairs."""
    spec, lay, sw, pool = built("long", gpu)
    for T in (3, 70):
        x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=T)
        out = mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu))
        _, _, want, bound = O.layer(spec, lay.experts, f64(x), idx, w)
        close(f64(bits(out)), want, bound, f"long T={T}")


def test_repeated_experts_of_a_token(gpu):
    """A routing that names one expert several times: each pair has its row."""
    spec, lay, sw, pool = built("clamped", gpu)
    for T in (1, 8, 30):
        x = acts(T, spec.hidden, 3)
        idx = np.full((T, spec.top_k), 2, np.int32)
        idx[:, 1] = 4
        w = np.full((T, spec.top_k), 0.25, np.float32)
        out = mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu))
        _, _, want, bound = O.layer(spec, lay.experts, f64(x), idx, w)
        close(f64(bits(out)), want, bound, f"repeated T={T}")


@pytest.mark.parametrize("T", [4, 40])
def test_nan_and_infinity_stay_with_their_token(gpu, T):
    spec, lay, sw, pool = built("swiglu", gpu)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=8)
    v = f64(x)
    x[1, 70], x[2, 3] = 0x7FC0, 0xFF80      # a NaN, minus infinity
    out = f64(bits(mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu))))
    assert np.isnan(out[1:3]).all()
    keep = np.r_[0, 3:T]
    _, _, want, bound = O.layer(spec, lay.experts, v, idx, w)
    close(out[keep], want[keep], bound[keep], "other tokens")


def test_zero_rows_and_no_tokens(gpu):
    import torch
    spec, lay, sw, pool = built("mlp", gpu)
    x = np.zeros((2, spec.hidden), np.uint16)
    idx, w = routing(spec, 2, 1)
    out = mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu))
    _, _, want, bound = O.layer(spec, lay.experts, f64(x), idx, w)
    close(f64(bits(out)), want, bound, "zero rows")
    out = mx.moe_forward(spec, pool, torch.zeros(0, spec.hidden, dtype=torch.bfloat16, device=gpu),
                         torch.zeros(0, spec.top_k, dtype=torch.int32, device=gpu),
                         torch.zeros(0, spec.top_k, device=gpu))
    assert tuple(out.shape) == (0, spec.hidden)


@pytest.mark.parametrize("T", [6, 48])
def test_a_row_does_not_depend_on_its_call(gpu, T):
    """The same token's row, whatever other pairs share the call (same kernel family): bit for bit."""
    spec, lay, sw, pool = built("clamped", gpu)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=21)
    flags = L.FWD_FORCE_DECODE if T <= 8 else L.FWD_FORCE_PREFILL
    xd, idd = to_dev_bits(x, gpu), dev(idx, gpu)
    rows = bits(mx.moe_forward(spec, pool, xd, idd, flags=flags))
    for t in (0, T // 2, T - 1):
        one = bits(mx.moe_forward(spec, pool, xd[t:t + 1], idd[t:t + 1], flags=flags))
        assert np.array_equal(one[0], rows[t])


@pytest.mark.parametrize("name", ["swiglu", "shared", "clamped", "mlp", "wide", "long"])
@pytest.mark.parametrize("T", [1, 3, 8, 9, 20, 64])
def test_every_kernel_family_gives_the_same_bits(gpu, name, T):
    spec, lay, sw, pool = built(name, gpu)
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=40 + T)
    if T == 8 and name == "clamped":
        idx[:, 1:] = 3                   # an expert with more pairs than a tile's smallest height
    xd, idd, wd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    kw = dict(shared=sw.shared, sgate=None if sg is None else dev(sg, gpu))
    fam = (L.FWD_FORCE_DECODE if T <= 8 else 0, L.FWD_FORCE_PREFILL)
    out = [bits(mx.moe_forward(spec, pool, xd, idd, wd, flags=f, **kw)) for f in fam]
    rows = [bits(mx.moe_forward(spec, pool, xd, idd, flags=f)) for f in fam]
    assert np.array_equal(*rows)
    assert np.array_equal(*out)


@pytest.mark.parametrize("name, proj", [("swiglu", "down_proj"), ("clamped", "gate_proj"), ("mlp", "fc1"), ("wide", "up_proj"),
                                        ("long", "down_proj")])
def test_short_and_long_lists_give_the_same_bits(gpu, name, proj):
    spec, pool, q, tok, ex, _, _ = _product(gpu, name, proj, 11, 200, seed=6)
    t, e = dev(tok, gpu), dev(ex, gpu)
    want = bits(mx.expert_product(spec, pool, q, t, e, proj))
    for a, b in ((0, 64), (3, 4), (10, 47), (0, 65), (72, 200)):
        got = bits(mx.expert_product(spec, pool, q, t[a:b].contiguous(), e[a:b].contiguous(), proj))
        assert np.array_equal(got, want[a:b])


@pytest.mark.parametrize("T", [4, 40])
def test_nan_passes_the_clamped_activation(gpu, T):
    spec, lay, sw, pool = built("clamped", gpu)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=9)
    x[2, 100] = 0x7F80
    out = f64(bits(mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu))))
    assert np.isnan(out[2]).all() and np.isfinite(out[np.r_[:2, 3:T]]).all()


# ------------------------------------------------------------------ as a program uses them
@pytest.mark.parametrize("T", [1, 5, 60])
def test_block_from_unquantized_weights(gpu, T):
    """Unquantized weights packed on the GPU, admitted to a pool, routed and run as a block whose
    activations are MXFP4; the shared expert beside them."""
    import torch
    spec = SHARED
    rng = np.random.default_rng(77)

    def weights(E, shared):
        es = spec.expert_spec(shared)
        return {p: torch.from_numpy(rng.standard_normal((E, c["scales"]["shape"][0], c["scales"]["shape"][1] * 32))
                                    .astype(np.float32) * 0.05).to(gpu).to(torch.bfloat16) for p, c in es.items()}
    packed = mx.pack_experts(spec, weights(spec.n_experts, False))
    shared = mx.pack_experts(spec, weights(1, True), shared=True)[0]
    pool = ExpertPool(0, spec, spec.n_experts).build()
    for e in range(spec.n_experts):
        pool.touch([e], [0])
        pool.admit_device(e, packed[e].data_ptr())
    sw = StreamingSwitchGLU(pool, None, shared=shared, activations="mxfp4")
    assert sw.refresh()
    router = to_dev_bits(F.f32_to_bf16_bits(rng.standard_normal((spec.n_experts, spec.hidden)).astype(np.float32) * 0.05), gpu)
    gate = to_dev_bits(F.f32_to_bf16_bits(rng.standard_normal(spec.hidden).astype(np.float32) * 0.05), gpu)
    moe = MoELayer(spec, router, sw, shared_gate_w=gate)
    x = acts(T, spec.hidden, 31)
    xd = to_dev_bits(x, gpu)
    out = moe(xd)
    idx, w, sg = moe.route(xd)
    blobs = [packed[e].cpu().numpy().tobytes() for e in range(spec.n_experts)]
    _, _, want, bound = O.layer(spec, blobs, f64(x), idx.cpu().numpy(), w.cpu().numpy(), shared.cpu().numpy().tobytes(),
                                sg.cpu().numpy())
    close(f64(bits(out)), want, bound, f"block T={T}")
    sw.activations = "bf16"      # the same layer with bf16 activations: near, not equal
    ref = f64(bits(moe(xd)))
    assert 1e-3 < np.linalg.norm(f64(bits(out)) - ref) / np.linalg.norm(ref) < 0.5
    pool.close()


@pytest.mark.parametrize("T", [2, 24])
def test_layer_is_its_parts(gpu, T):
    """quantize, the gate and up products, the activation, quantize, the down product: the layer's rows,
    where the parts' bf16 roundings allow."""
    import torch
    spec, lay, sw, pool = built("swiglu", gpu)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=5)
    xd = to_dev_bits(x, gpu)
    tok = torch.arange(T, device=gpu, dtype=torch.int32).repeat_interleave(spec.top_k)
    ex = dev(idx.reshape(-1), gpu)
    q = mx.quantize(xd)
    g = mx.expert_product(spec, pool, q, tok, ex, "gate_proj").float()
    u = mx.expert_product(spec, pool, q, tok, ex, "up_proj").float()
    own = torch.arange(T * spec.top_k, device=gpu, dtype=torch.int32)
    y = mx.expert_product(spec, pool, mx.quantize(g * torch.sigmoid(g) * u), own, ex, "down_proj")
    rows = mx.moe_forward(spec, pool, xd, ex.view(T, -1)).view(T * spec.top_k, -1)
    # the products' bf16 roundings move an element of h by up to 2^-7 of it, and so its code by a step
    # now and then: a whole step (a third of a value) for about one in 2^7 / 4 elements
    assert ((y - rows).float().norm() / rows.float().norm()).item() < 0.34 * (4 / 2 ** 7) ** 0.5 + 2.0 ** -6


@pytest.mark.parametrize("T", [5, 40])
def test_bounded_pool_and_host_served(gpu, T):
    """A pool of three slots (spans over the step's experts) and one whose misses the kernels read from
    pinned host memory give the resident layer's bits."""
    import torch
    spec, lay, sw, pool = built("shared", gpu)
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=13)
    xd, idd, wd, sgd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), dev(sg, gpu)
    want_rows = bits(sw(xd, idd))
    want = bits(sw.forward_combined(xd, idd, wd, sgd))
    for host in (False, True):
        store = HostStore()
        store.add_layer(0, lay.experts)
        p = ExpertPool(0, spec, 3).build()
        s = StreamingSwitchGLU(p, PinnedFetcher(store), shared=sw.shared, host_served=host, activations="mxfp4")
        for _ in range(3):
            assert np.array_equal(bits(s(xd, idd)), want_rows)
            assert np.array_equal(bits(s.forward_combined(xd, idd, wd, sgd)), want)
        assert host or s.chunked_calls > 0
        torch.cuda.synchronize()
        p.close()


@pytest.mark.parametrize("T", [3, 20])
def test_absent_expert_is_nan_and_reported(gpu, T):
    import torch
    spec, lay, _, _ = built("swiglu", gpu)
    store = HostStore()
    store.add_layer(0, lay.experts)
    pool = ExpertPool(0, spec, 5).build()
    for e in range(5):                   # expert 5 stays absent
        pool.touch([e], [0])
        pool.admit(e, store.region(0, e))
    pool.g2s_device(torch.cuda.current_stream().cuda_stream)
    x = acts(T, spec.hidden, 2)
    idx = np.tile(np.int32([0, 3]), (T, 1))
    idx[1, 1] = 5
    w = np.full((T, 2), 0.5, np.float32)
    xd, idd = to_dev_bits(x, gpu), dev(idx, gpu)
    rows = f64(bits(mx.moe_forward(spec, pool, xd, idd)))
    with pytest.raises(L.BrxError, match="expert 5"):
        pool.device.check()
    out = f64(bits(mx.moe_forward(spec, pool, xd, idd, dev(w, gpu))))
    with pytest.raises(L.BrxError, match="expert 5"):
        pool.device.check()
    q = mx.quantize(xd)
    tok = torch.arange(T, device=gpu, dtype=torch.int32)
    y = f64(bits(mx.expert_product(spec, pool, q, tok, idd[:, 1].contiguous(), "gate_proj")))
    with pytest.raises(L.BrxError, match="expert 5"):
        pool.device.check()
    keep = np.r_[0, 2:T]
    assert np.isnan(rows[1, 1]).all() and np.isfinite(rows[1, 0]).all() and np.isfinite(rows[keep]).all()
    assert np.isnan(out[1]).all() and np.isfinite(out[keep]).all()
    assert np.isnan(y[1]).all() and np.isfinite(y[keep]).all()
    pool.device.check()
    pool.close()


@pytest.mark.parametrize("T", [2, 40])
def test_two_streams(gpu, T):
    """Calls on two streams at once, each with scratch of its own."""
    import torch
    spec, lay, sw, pool = built("clamped", gpu)
    ins, want = [], []
    for s in range(2):
        x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=50 + s)
        ins.append((to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)))
        want.append(bits(mx.moe_forward(spec, pool, *ins[-1])))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for s in range(2):
            got[s].append(mx.moe_forward(spec, pool, *ins[s], stream=streams[s]))
    torch.cuda.synchronize()
    for s in range(2):
        for g in got[s]:
            assert np.array_equal(bits(g), want[s])


@pytest.mark.parametrize("name, T", [("shared", 1), ("shared", 33), ("clamped", 7), ("mlp", 70)])
def test_combine_of_float32_rows(gpu, name, T):
    """The pairs' float32 rows and their combine: the layer call's sums, bit for bit; rounded, its bf16 rows."""
    import torch
    spec, lay, sw, pool = built(name, gpu)
    E, k, H = spec.n_experts, spec.top_k, spec.hidden
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=80 + T)
    xd, idd, wd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    sgd = None if sg is None else dev(sg, gpu)
    want = bits(mx.moe_forward(spec, pool, xd, idd, wd, shared=sw.shared, sgate=sgd))
    tok = torch.arange(T, dtype=torch.int32, device=gpu)
    for f in (0, L.FWD_FORCE_PREFILL):
        y = torch.empty((T * k, H), device=gpu)
        mx.forward_pairs(spec, pool, xd, tok.repeat_interleave(k), idd.view(-1), None, y, f)
        ysh = None
        if sw.shared is not None:
            ysh = torch.empty((T, H), device=gpu)
            mx.forward_pairs(spec, pool, xd, tok, torch.full_like(tok, E), None, ysh, f, shared=sw.shared)
        out = torch.empty((T, H), dtype=torch.bfloat16, device=gpu)
        mx.combine(spec, y, wd, out, ysh, sgd)
        assert np.array_equal(bits(out), want)
        assert np.array_equal(bits(y.bfloat16()), bits(mx.moe_forward(spec, pool, xd, idd)).reshape(T * k, H))
    for kw, what in ((dict(y_routed=y.bfloat16()), "y_routed"), (dict(w=wd[:0]), "w must"), (dict(out=out.float()), "out"),
                     (dict(y_shared=y[:0]), "y_shared"), (dict(sgate=wd.view(-1)[:0]), "sgate")):
        with pytest.raises(ValueError, match=what):
            mx.combine(**dict(dict(spec=spec, y_routed=y, w=wd, out=out), **kw))
    with pytest.raises(L.BrxError, match="gate"):
        mx.combine(spec, y, wd, out, torch.zeros((T, H), device=gpu))


def test_a_given_stream_has_the_whole_call(gpu):
    """Given a stream, a call takes its memory there (not a block that the current stream's queued work may
    still read), and copies a strided x there, behind the work that makes it."""
    import torch
    spec, lay, sw, pool = built("swiglu", gpu)
    s = torch.cuda.Stream()
    x = to_dev_bits(acts(64, spec.hidden, 3), gpu)
    idx, w = routing(spec, 64, 3)
    idd, wd = dev(idx, gpu), dev(w, gpu)
    want = bits(mx.moe_forward(spec, pool, x, idd, wd))
    rows = mx.quantize(x)
    torch.cuda.synchronize()
    calls = {"quantize": lambda: mx.quantize(x, stream=s).codes,
             "dequantize": lambda: mx.dequantize(rows, stream=s),
             "forward": lambda: mx.moe_forward(spec, pool, x, idd, wd, stream=s)}
    for what, call in calls.items():
        got = call()
        torch.cuda.synchronize()
        size = got.numel() * got.element_size()
        del got
        torch.cuda.empty_cache()
        freed = torch.empty(size, dtype=torch.uint8, device=gpu)
        at = freed.data_ptr()
        del freed
        assert call().data_ptr() != at, what
        torch.cuda.synchronize()
    late = torch.zeros((64, 2 * spec.hidden), dtype=torch.bfloat16, device=gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        late[:, :spec.hidden] = x
    got = mx.moe_forward(spec, pool, late[:, :spec.hidden], idd, wd, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert np.array_equal(bits(got), want)


@pytest.mark.parametrize("T", [3, 20, 90])
def test_pairs_with_the_shared_expert(gpu, T):
    """The pairs form with the shared expert's id among them, in shuffled rows: the layer call's rows and the
    shared expert's, whichever kernels run; rows no pair names stay."""
    import torch
    spec, lay, sw, pool = built("shared", gpu)
    E, k = spec.n_experts, spec.top_k
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=70 + T)
    xd = to_dev_bits(x, gpu)
    tok = np.concatenate([np.repeat(np.arange(T), k), np.arange(T)]).astype(np.int32)
    ex = np.concatenate([idx.reshape(-1), np.full(T, E)]).astype(np.int32)
    row = np.random.default_rng(T).permutation(tok.size + 5)[:tok.size].astype(np.int32)
    got = []
    for f in (0, L.FWD_FORCE_PREFILL) + ((L.FWD_FORCE_DECODE,) if T <= 8 else ()):
        y = torch.full((tok.size + 5, spec.hidden), 3.0, dtype=torch.bfloat16, device=gpu)
        mx.forward_pairs(spec, pool, xd, dev(tok, gpu), dev(ex, gpu), dev(row, gpu), y, f, shared=sw.shared)
        got.append(bits(y))
        assert np.array_equal(got[-1], got[0])
    assert (f64(np.delete(got[0], row, 0)) == 3.0).all()
    routed = bits(mx.moe_forward(spec, pool, xd, dev(idx, gpu))).reshape(T * k, spec.hidden)
    assert np.array_equal(got[0][row[:T * k]], routed)
    # weight 0 for the routed experts leaves the shared expert's rows (times one)
    zero, one = torch.zeros((T, k), device=gpu), torch.ones(T, device=gpu)
    alone = bits(mx.moe_forward(spec, pool, xd, dev(idx, gpu), zero, shared=sw.shared, sgate=one))
    assert np.array_equal(f64(got[0][row[T * k:]]), f64(alone))


@pytest.mark.parametrize("T", [2, 40])
def test_refill_waits_for_a_resident_pools_calls(gpu, T):
    """A slot is refilled behind a queued call that reads it, on a copy stream; the pool's sync waits for the
    call; a bf16 forward and an MXFP4 call on two streams are both waited for."""
    import torch
    lay = make_layer(SWIGLU, seed=77, expert_std=0.05)
    _, sw, pool, _ = build_gpu_layer(lay, gpu)
    spec, lib, h = lay.spec, L.load(), pool.device.handle
    pool.g2s_device(torch.cuda.current_stream().cuda_stream)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=61)
    xd, idd, wd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    old = bits(mx.moe_forward(spec, pool, xd, idd, wd))
    plain = bits(layer_forward(spec, pool, xd, idd, wd))
    blobs = [bytes_dev(b, gpu) for b in lay.experts]
    slots = pool.g2s
    torch.cuda.synchronize()
    run, other, copy = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    for both in (False, True):
        with torch.cuda.stream(other):
            if both:
                torch.cuda._sleep(40_000_000)
                p16 = layer_forward(spec, pool, xd, idd, wd)
        with torch.cuda.stream(run):
            torch.cuda._sleep(20_000_000)
            got = mx.moe_forward(spec, pool, xd, idd, wd)
        for e in range(spec.n_experts):      # every expert's slot takes the next expert's bytes
            b = blobs[(e + 1) % spec.n_experts]
            L.check(lib.brx_pool_refill_from_device_async(h, int(slots[e]), b.data_ptr(), b.numel(), copy.cuda_stream))
        torch.cuda.synchronize()
        assert np.array_equal(bits(got), old)
        assert not both or np.array_equal(bits(p16), plain)
        assert not np.array_equal(bits(mx.moe_forward(spec, pool, xd, idd, wd)), old)
        for e in range(spec.n_experts):
            L.check(lib.brx_pool_refill_from_device_async(h, int(slots[e]), blobs[e].data_ptr(), blobs[e].numel(), copy.cuda_stream))
        assert np.array_equal(bits(mx.moe_forward(spec, pool, xd, idd, wd)), old)
    with torch.cuda.stream(run):
        torch.cuda._sleep(20_000_000)
        mx.moe_forward(spec, pool, xd, idd, wd)
    L.check(lib.brx_pool_sync(h))
    assert run.query()
    pool.device.check()
    pool.close()


@pytest.mark.parametrize("T", [3, 12, 150])
def test_sums_and_rows_of_one_call(gpu, T):
    """Both outputs at once, into tensors given: those of a call each."""
    import torch
    spec, lay, sw, pool = built("shared", gpu)
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=33)
    xd, idd, wd, sgd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), dev(sg, gpu)
    kw = dict(shared=sw.shared, sgate=sgd)
    out = torch.empty((T, spec.hidden), dtype=torch.bfloat16, device=gpu)
    rows = torch.empty((T, spec.top_k, spec.hidden), dtype=torch.bfloat16, device=gpu)
    assert mx.moe_forward(spec, pool, xd, idd, wd, out=out, y_unreduced=rows, **kw) is out
    assert np.array_equal(bits(out), bits(mx.moe_forward(spec, pool, xd, idd, wd, **kw)))
    assert np.array_equal(bits(rows), bits(mx.moe_forward(spec, pool, xd, idd)))
    with pytest.raises(ValueError, match="y_rows"):
        mx.forward_pairs(spec, pool, xd, idd.view(-1)[:T], idd.view(-1)[:T], None, rows[:, 0].half().contiguous(), 0)


@pytest.mark.parametrize("T", [1, 8, 30])
def test_captured_graphs(gpu, T):
    """Two captured layers (rows quantised and read back beside them), replayed in turn and with eager
    calls between, each replay against the eager result for the inputs of the moment."""
    import torch
    spec, lay, sw, pool = built("shared", gpu)
    xs = [torch.zeros((T, spec.hidden), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    ids = [torch.zeros((T, spec.top_k), dtype=torch.int32, device=gpu) for _ in range(2)]
    ws = [torch.ones((T, spec.top_k), device=gpu) for _ in range(2)]
    sg = torch.full((T,), 0.5, device=gpu)
    graphs, outs = [], []

    def call(s):
        return (mx.moe_forward(spec, pool, xs[s], ids[s], ws[s], shared=sw.shared, sgate=sg),
                mx.dequantize(mx.quantize(xs[s]), torch.float32))
    for s in range(2):
        call(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = call(s)
        graphs.append(g)
        outs.append(o)
    for rnd in range(4):
        for s in range(2):
            x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=90 + 2 * rnd + s)
            xs[s].copy_(to_dev_bits(x, gpu))
            ids[s].copy_(dev(idx, gpu))
            ws[s].copy_(dev(w, gpu))
        for s in range(2):
            graphs[s].replay()
        eager = [call(s) for s in range(2)]
        torch.cuda.synchronize()
        for s in range(2):
            assert np.array_equal(bits(outs[s][0]), bits(eager[s][0])), (rnd, s)
            assert torch.equal(outs[s][1], eager[s][1]), (rnd, s)


def test_layer_refusals(gpu):
    import torch
    spec, lay, sw, pool = built("swiglu", gpu)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, 4, seed=1)
    x, idx, w = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    call = lambda **kw: mx.moe_forward(**dict(dict(spec=spec, pool=pool, x=x, idx=idx, w=w), **kw))   # noqa: E731
    for kw, what in ((dict(x=x.float()), "bfloat16"), (dict(x=x[:, :64]), "bfloat16"), (dict(idx=idx[:3]), "idx"),
                     (dict(idx=idx.long()), "idx"), (dict(w=w.half()), "w must"), (dict(w=w[:, :1]), "w must"),
                     (dict(shared=torch.zeros(8, dtype=torch.uint8, device=gpu)), "shared"),
                     (dict(out=torch.zeros(4, 320, device=gpu)), "out and"), (dict(idx=idx.cpu()), "on the GPU"),
                     (dict(sgate=torch.zeros(3, device=gpu)), "sgate")):
        with pytest.raises(ValueError, match=what):
            call(**kw)
    with pytest.raises(L.BrxError, match="flags"):
        call(flags=L.FWD_PHASE_A)
    with pytest.raises(L.BrxError, match="exclusive"):
        call(flags=3)
    with pytest.raises(L.BrxError, match="descriptor differs"):
        call(spec=small(spec, route_scale=2.0))
    sspec, slay, ssw, spool = built("shared", gpu)
    sx, sidx, swt, _ = _layer_inputs(sspec, slay, gpu, 2, seed=1)
    with pytest.raises(L.BrxError, match="gate"):
        mx.moe_forward(sspec, spool, to_dev_bits(sx, gpu), dev(sidx, gpu), dev(swt, gpu), shared=ssw.shared)
    d = spec.desc()
    lib = L.load()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    out = torch.zeros_like(x)

    def raw(xp=x.data_ptr(), ip=idx.data_ptr(), wp=w.data_ptr(), T=4, op=out.data_ptr(), p=ws.data_ptr(), n=ws.numel(),
            flags=0):
        return lib.brx_mx_moe_forward(C.byref(d), pool.device.handle, xp, ip, wp, None, None, T, op, None, flags, p, n, None)
    for kw in (dict(xp=None), dict(xp=x.data_ptr() + 2), dict(ip=None), dict(wp=None), dict(op=None), dict(T=-1),
               dict(T=65536), dict(op=out.data_ptr() + 2), dict(p=None), dict(n=100)):
        assert raw(**kw) == L.BRX_EINVAL, kw
    assert raw() == 0
    torch.cuda.synchronize()

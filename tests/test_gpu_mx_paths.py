"""The MXFP4 operators' kernels past the few-pair ones, and the limits of their calls, on the GPU."""
import ctypes as C

import numpy as np
import pytest

from bigrig_amd import lib as L
from bigrig_amd import mx
from bigrig_amd.layer import StreamingSwitchGLU
from bigrig_amd.pool import ExpertPool, HostStore, PinnedFetcher
from bigrig_amd.spec import E256_SHARED, GPT_OSS_120B, QWEN3_30B_A3B
from tests import mx_oracle as O
from tests.gpu_util import bits, build_gpu_layer, to_dev_bits
from tests.helpers import make_layer, small
from tests.test_gpu_mx import MX, _layer_inputs, _product, acts, built, close, dev, f64

pytestmark = pytest.mark.gpu

# More experts than a wave has lanes, than a byte counts, and the most there are (the shared one's id is 512).
E100 = small(QWEN3_30B_A3B, quant=MX, hidden=64, inter=64, n_experts=100, top_k=4)
E300 = small(E256_SHARED, quant=MX, hidden=128, inter=64, shared_inter=128, n_experts=300, top_k=8)
E512 = small(E256_SHARED, quant=MX, hidden=64, inter=64, shared_inter=64, n_experts=512, top_k=8)
MANY = {"e100": E100, "e300": E300, "e512": E512}
# the widest input: the few-pair kernels' LDS rows of 16 chunks, up to 16 pairs of them
TALL = small(GPT_OSS_120B, hidden=8192, inter=128, n_experts=4, top_k=2)
_BUILT = {}


def _many(name, gpu):
    import torch
    if name not in _BUILT:
        spec = TALL if name == "tall" else MANY[name]
        lay = make_layer(spec, seed=700 + spec.n_experts, bank=None if name == "tall" else 23, expert_std=0.05)
        _, sw, pool, _ = build_gpu_layer(lay, gpu)
        sw.activations = "mxfp4"
        pool.g2s_device(torch.cuda.current_stream().cuda_stream)
        _BUILT[name] = (spec, lay, sw, pool)
    return _BUILT[name]


def _spread(spec, T, seed):
    """A routing whose ids are spread over all experts, the first, the last and the borders of 64 and 256 among
    them, each token's distinct; popular ones repeat over the tokens."""
    rng = np.random.default_rng(seed)
    E, k = spec.n_experts, spec.top_k
    edge = [e for e in (0, 63, 64, 127, 128, 255, 256, E - 1) if e < E]
    idx = np.stack([rng.choice(E, k, replace=False) for _ in range(T)])
    for t in range(0, T, 2):
        e = edge[(t // 2) % len(edge)]
        if e not in idx[t]:
            idx[t, rng.integers(0, k)] = e
    w = rng.random((T, k), dtype=np.float32) + 0.1
    return idx.astype(np.int32), w / w.sum(1, keepdims=True)


# The lines between the kernels: 8 tokens and 64 pairs, 64 tokens, 128 and 256 pairs (k_mx.hip, mx_path); few pairs a
# lane, two, a bucketing, the grouped GEMM.
@pytest.mark.parametrize("name, T", [("e100", 1), ("e100", 8), ("e100", 16), ("e100", 17), ("e100", 32), ("e100", 33),
                                     ("e100", 64), ("e100", 65), ("e300", 1), ("e300", 8), ("e300", 9), ("e300", 16),
                                     ("e300", 17), ("e300", 32), ("e300", 33), ("e512", 1), ("e512", 8), ("e512", 16),
                                     ("e512", 30), ("e512", 100)])
def test_layers_of_many_experts(gpu, name, T):
    spec, lay, sw, pool = _many(name, gpu)
    x = acts(T, spec.hidden, T)
    idx, w = _spread(spec, T, 3 * T)
    xd, idd, wd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    kw, sg = {}, None
    if lay.shared is not None:
        sg = np.random.default_rng(T).random(T, dtype=np.float32)
        kw = dict(shared=sw.shared, sgate=dev(sg, gpu))
    y, dy, want, bound = O.layer(spec, lay.experts, f64(x), idx, w, lay.shared, sg)
    rows = bits(mx.moe_forward(spec, pool, xd, idd))
    out = bits(mx.moe_forward(spec, pool, xd, idd, wd, **kw))
    close(f64(rows), y, dy, f"{name} rows T={T}")
    close(f64(out), want, bound, f"{name} T={T}")
    assert np.array_equal(bits(mx.moe_forward(spec, pool, xd, idd, flags=L.FWD_FORCE_PREFILL)), rows)
    assert np.array_equal(bits(mx.moe_forward(spec, pool, xd, idd, wd, flags=L.FWD_FORCE_PREFILL, **kw)), out)


@pytest.mark.parametrize("name", ["e100", "e300", "e512"])
@pytest.mark.parametrize("P", [1, 8, 64, 65, 128, 129, 600])
def test_pair_lists_of_many_experts(gpu, name, P):
    """The pairs form (the shared expert's id, which is the number of experts, among them) and the expert product."""
    import torch
    spec, lay, sw, pool = _many(name, gpu)
    E, T = spec.n_experts, 11
    x = acts(T, spec.hidden, P)
    rng = np.random.default_rng(P)
    ex = rng.integers(0, E, P).astype(np.int32)
    ex[::5] = E - 1
    if P > 2:
        ex[1], ex[2] = 0, min(64, E - 1)
    tok = rng.integers(0, T, P).astype(np.int32)
    xd = to_dev_bits(x, gpu)
    xq = O.held(f64(x))
    ex_sh = ex.copy()
    if lay.shared is not None:
        ex_sh[3::4] = E
    want, bound = np.zeros((P, spec.hidden)), np.zeros((P, spec.hidden))
    up, dup = np.zeros((P, spec.inter)), np.zeros((P, spec.inter))
    for e in np.unique(np.concatenate([ex, ex_sh])):
        i = np.flatnonzero(ex_sh == e)
        if i.size:
            want[i], bound[i] = O.expert_rows(spec, lay.shared if e == E else lay.experts[e], xq[tok[i]], e == E)
        i = np.flatnonzero(ex == e)
        if i.size:
            up[i], dup[i] = O.product(*O.weights(spec, lay.experts[e], "up_proj"), xq[tok[i]])
    row = rng.permutation(P + 3)[:P].astype(np.int32)
    y = torch.full((P + 3, spec.hidden), 5.0, dtype=torch.bfloat16, device=gpu)
    mx.forward_pairs(spec, pool, xd, dev(tok, gpu), dev(ex_sh, gpu), dev(row, gpu), y, 0, shared=sw.shared)
    close(f64(bits(y))[row], want, bound + 2.0 ** -8 * (np.abs(want) + bound), f"{name} P={P}")
    assert (f64(np.delete(bits(y), row, 0)) == 5.0).all()
    got = mx.expert_product(spec, pool, mx.quantize(xd), dev(tok, gpu), dev(ex, gpu), "up_proj")
    close(f64(bits(got)), up, dup + 2.0 ** -8 * (np.abs(up) + dup), f"{name} product P={P}")


@pytest.mark.parametrize("T", [1, 8, 20, 70])
def test_layer_of_the_widest_input(gpu, T):
    """Rows of 16 chunks; at 8 tokens one expert has 8 pairs of them in LDS, at 20 an entry has 16."""
    spec, lay, sw, pool = _many("tall", gpu)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=T)
    idx[:, 0], idx[:, 1] = 2, np.arange(T) % 2
    xd, idd, wd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    out = bits(mx.moe_forward(spec, pool, xd, idd, wd))
    _, _, want, bound = O.layer(spec, lay.experts, f64(x), idx, w)
    close(f64(out), want, bound, f"widest T={T}")
    assert np.array_equal(bits(mx.moe_forward(spec, pool, xd, idd, wd, flags=L.FWD_FORCE_PREFILL)), out)


# ------------------------------------------------------------------ what few-pair calls are tested for, in the GEMM
@pytest.mark.parametrize("name", ["swiglu", "clamped", "shared", "mlp"])
@pytest.mark.parametrize("T", [20, 45, 150])        # (tiles of 16, 32 and 64 pairs)
def test_nan_stays_with_its_token_in_the_gemm(gpu, name, T):
    spec, lay, sw, pool = built(name, gpu)
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=18)
    v = f64(x)
    x[1, 10], x[2, 3], x[T - 1, spec.hidden - 1] = 0x7FC0, 0xFF80, 0x7F80      # a NaN, both infinities
    kw = {} if sg is None else dict(shared=sw.shared, sgate=dev(sg, gpu))
    xd, idd = to_dev_bits(x, gpu), dev(idx, gpu)
    out = f64(bits(mx.moe_forward(spec, pool, xd, idd, dev(w, gpu), flags=L.FWD_FORCE_PREFILL, **kw)))
    rows = f64(bits(mx.moe_forward(spec, pool, xd, idd, flags=L.FWD_FORCE_PREFILL)))
    bad = np.r_[1, 2, T - 1]
    assert np.isnan(out[bad]).all() and np.isnan(rows[bad]).all()
    keep = np.r_[0, 3:T - 1]
    y, dy, want, bound = O.layer(spec, lay.experts, v, idx, w, lay.shared, sg)
    close(out[keep], want[keep], bound[keep], "other tokens")
    close(rows[keep], y[keep], dy[keep], "other tokens' rows")


@pytest.mark.parametrize("P", [40, 200, 500])
def test_nan_stays_with_its_row_in_a_product(gpu, P):
    spec, pool, q, tok, ex, want, bound = _product(gpu, "swiglu", "down_proj", 30, P, seed=P)
    t = int(tok[0])                       # (a token that some pair names)
    q.scales[t, 1] = 255
    got = f64(bits(mx.expert_product(spec, pool, q, dev(tok, gpu), dev(ex, gpu), "down_proj")))
    assert np.isnan(got[tok == t]).all()
    close(got[tok != t], want[tok != t], bound[tok != t], f"other rows P={P}")


@pytest.mark.parametrize("T", [20, 45, 150])
def test_absent_expert_in_the_gemm(gpu, T):
    """Gate/up, down and one projection of an expert that is in no slot: its pairs NaN, the others theirs."""
    import torch
    spec, lay, _, _ = built("swiglu", gpu)
    store = HostStore()
    store.add_layer(0, lay.experts)
    pool = ExpertPool(0, spec, 5).build()
    for e in range(5):                   # expert 5 stays absent
        pool.touch([e], [0])
        pool.admit(e, store.region(0, e))
    pool.g2s_device(torch.cuda.current_stream().cuda_stream)
    x, idx, w, _ = _layer_inputs(spec, lay, gpu, T, seed=5)
    gone = (idx == 5).any(1)
    assert gone.any() and not gone.all()
    xd, idd, wd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    y, dy, want, bound = O.layer(spec, lay.experts, f64(x), idx, w)
    for f in (0, L.FWD_FORCE_PREFILL):
        rows = f64(bits(mx.moe_forward(spec, pool, xd, idd, flags=f)))
        with pytest.raises(L.BrxError, match="expert 5"):
            pool.device.check()
        out = f64(bits(mx.moe_forward(spec, pool, xd, idd, wd, flags=f)))
        with pytest.raises(L.BrxError, match="expert 5"):
            pool.device.check()
        assert np.isnan(rows[idx == 5]).all() and np.isnan(out[gone]).all()
        close(rows[idx != 5], y[idx != 5], dy[idx != 5], "other rows")
        close(out[~gone], want[~gone], bound[~gone], "other tokens")
    q, tok = mx.quantize(xd), torch.arange(T, device=gpu, dtype=torch.int32).repeat_interleave(2)
    pairs = torch.cat([idd.view(-1)] * 4)
    got = f64(bits(mx.expert_product(spec, pool, q, torch.cat([tok] * 4), pairs, "gate_proj")))
    with pytest.raises(L.BrxError, match="expert 5"):
        pool.device.check()
    away = np.tile(idx.reshape(-1) == 5, 4)
    assert np.isnan(got[away]).all() and np.isfinite(got[~away]).all()
    pool.device.check()
    pool.close()


@pytest.mark.parametrize("host", [False, True])
def test_bounded_pools_on_the_gemm(gpu, host):
    """Spans of three experts, and experts read from pinned host memory, in calls of 450 pairs: the resident
    layer's bits."""
    import torch
    spec, lay, sw, pool = built("shared", gpu)
    T = 150
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=14)
    xd, idd, wd, sgd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), dev(sg, gpu)
    want_rows, want = bits(sw(xd, idd)), bits(sw.forward_combined(xd, idd, wd, sgd))
    store = HostStore()
    store.add_layer(0, lay.experts)
    p = ExpertPool(0, spec, 3).build()
    s = StreamingSwitchGLU(p, PinnedFetcher(store), shared=sw.shared, host_served=host, activations="mxfp4")
    for _ in range(4):                    # (host-served: residency moves behind the calls)
        assert np.array_equal(bits(s(xd, idd)), want_rows)
        assert np.array_equal(bits(s.forward_combined(xd, idd, wd, sgd)), want)
    assert host or s.chunked_calls == 8
    torch.cuda.synchronize()
    p.close()


def test_repeated_experts_in_the_gemm(gpu):
    spec, lay, sw, pool = built("clamped", gpu)
    T = 110
    x = acts(T, spec.hidden, 3)
    idx = np.full((T, spec.top_k), 2, np.int32)
    idx[:, 1], idx[::3, 3] = 4, 0
    w = np.full((T, spec.top_k), 0.25, np.float32)
    out = mx.moe_forward(spec, pool, to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu))
    _, _, want, bound = O.layer(spec, lay.experts, f64(x), idx, w)
    close(f64(bits(out)), want, bound, "repeated")


@pytest.mark.parametrize("T", [66, 300])
def test_two_streams_and_graphs_on_the_gemm(gpu, T):
    """Calls on two streams at once, then two captured layers and products replayed in turn between eager calls:
    every one the lone call's bits."""
    import torch
    spec, lay, sw, pool = built("shared", gpu)
    tok = torch.arange(T, device=gpu, dtype=torch.int32).repeat_interleave(spec.top_k)
    ins = []
    for s in range(6):
        x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=150 + s)
        ins.append((to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), dev(sg, gpu)))

    def call(a):
        out = mx.moe_forward(spec, pool, a[0], a[1], a[2], shared=sw.shared, sgate=a[3])
        return out, mx.expert_product(spec, pool, mx.quantize(a[0]), tok, a[1].view(-1), "up_proj")
    want = [tuple(bits(t) for t in call(a)) for a in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(call(ins[s]))
    torch.cuda.synchronize()
    for s in range(2):
        for g in got[s]:
            assert all(np.array_equal(bits(a), b) for a, b in zip(g, want[s]))
    own = [[t.clone() for t in ins[s]] for s in range(2)]
    graphs, outs = [], []
    for s in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(own[s]))
        graphs.append(g)
    for rnd in range(3):
        use = [ins[2 * rnd], ins[2 * rnd + 1]]
        for s in range(2):
            for a, b in zip(own[s], use[s]):
                a.copy_(b)
        for s in range(2):
            graphs[s].replay()
        eager = call(ins[0])
        torch.cuda.synchronize()
        for s in range(2):
            for a, b in zip(outs[s], want[2 * rnd + s]):
                assert np.array_equal(bits(a), b), (rnd, s)
        assert all(np.array_equal(bits(a), b) for a, b in zip(eager, want[0]))


def test_pairs_of_rows_past_32_bit_offsets_are_refused(gpu):
    """2^20 rows of 8192 values have 4 GB of codes: the pairs form refuses them as the product does, before it
    looks at the rows (the pointers are a small tensor's)."""
    import torch
    spec = small(GPT_OSS_120B, hidden=8192, inter=64, n_experts=2, top_k=1)
    _, _, pool, _ = build_gpu_layer(make_layer(spec, seed=5, expert_std=0.05), gpu)
    x = torch.zeros(1 << 16, dtype=torch.uint8, device=gpu)
    pair = torch.zeros(1, dtype=torch.int32, device=gpu)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    d, lib = spec.desc(), L.load()
    for T in (1 << 20, (1 << 31) - 1):
        rc = lib.brx_mx_moe_forward_pairs(C.byref(d), pool.device.handle, x.data_ptr(), T, pair.data_ptr(), pair.data_ptr(),
                                          None, 1, 1, None, x.data_ptr(), L.DT_BF16, 0, ws.data_ptr(), ws.numel(), None)
        assert rc == L.BRX_EINVAL and "2^32 - 256" in lib.brx_last_error().decode()
        rc = lib.brx_mx_expert_product(C.byref(d), pool.device.handle, x.data_ptr(), x.data_ptr(), T, pair.data_ptr(),
                                       pair.data_ptr(), None, 1, 1, 0, x.data_ptr(), ws.data_ptr(), ws.numel(), None)
        assert rc == L.BRX_EINVAL and "2^32 - 256" in lib.brx_last_error().decode()
    torch.cuda.synchronize()
    pool.close()

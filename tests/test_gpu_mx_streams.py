"""Layers of MXFP4 experts on streams of the caller's."""
import numpy as np
import pytest

from bigrig_amd import formats as F
from bigrig_amd import lib as L
from bigrig_amd import mx
from bigrig_amd.layer import MoELayer, StreamingSwitchGLU
from bigrig_amd.pool import ExpertPool, HostStore, PinnedFetcher
from tests.gpu_util import bits, build_gpu_layer, bytes_dev, to_dev_bits
from tests.helpers import make_layer
from tests.test_gpu_mx import SHARED, SWIGLU, _layer_inputs, dev, layer_forward

pytestmark = pytest.mark.gpu


def _switch(lay, gpu, kind, activations):
    """(switch, pool) over every expert, three slots, or three slots and host backing."""
    import torch
    if kind == "resident":
        _, sw, pool, _ = build_gpu_layer(lay, gpu)
        sw.activations = activations
        assert sw.refresh()
        torch.cuda.synchronize()
        return sw, pool
    store = HostStore()
    store.add_layer(0, lay.experts)
    pool = ExpertPool(0, lay.spec, 3).build()
    shared = torch.frombuffer(bytearray(lay.shared), dtype=torch.uint8).to(gpu)
    return StreamingSwitchGLU(pool, PinnedFetcher(store), shared=shared, host_served=kind == "host",
                              activations=activations), pool


def _scribble(gpu):
    """Every size of block the current stream's allocator may hand out, overwritten on the current stream."""
    import torch
    held = [torch.full((n,), 0xFF, dtype=torch.uint8, device=gpu) for n in (512, 1024, 4096, 16384, 65536, 1 << 18, 1 << 20)
            for _ in range(12)]
    del held


@pytest.mark.parametrize("activations", ["bf16", "mxfp4"])
@pytest.mark.parametrize("kind", ["resident", "bounded", "host"])
@pytest.mark.parametrize("T", [3, 90])
def test_layer_calls_on_a_given_stream(gpu, kind, activations, T):
    """The switch's and the block's calls on a side stream with work ahead of them, their inputs freed and the
    current stream's memory overwritten as soon as they return: the current stream's bits."""
    import torch
    lay = make_layer(SHARED, seed=91, expert_std=0.05)
    spec = lay.spec
    sw, pool = _switch(lay, gpu, kind, activations)
    rng = np.random.default_rng(7)
    router = to_dev_bits(F.f32_to_bf16_bits(rng.standard_normal((spec.n_experts, spec.hidden)).astype(np.float32) * 0.05), gpu)
    gate = to_dev_bits(F.f32_to_bf16_bits(rng.standard_normal(spec.hidden).astype(np.float32) * 0.05), gpu)
    moe = MoELayer(spec, router, sw, shared_gate_w=gate)
    x, idx, w, sg = _layer_inputs(spec, lay, gpu, T, seed=19 + T)
    xd, idd, wd, sgd = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), dev(sg, gpu)
    calls = {"rows": lambda *a, **k: sw(a[0], a[1], **k), "combined": lambda *a, **k: sw.forward_combined(*a, **k),
             "block": lambda *a, **k: moe(a[0], **k)}
    want = {n: bits(f(xd, idd, wd, sgd)) for n, f in calls.items()}
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for n, f in calls.items():
        for strided in (False, True):
            a = [t.clone() for t in (xd, idd, wd, sgd)]
            if strided and n != "combined":       # (its tokens are taken as they are)
                a[0] = torch.cat([xd, xd], 1)[:, :spec.hidden]
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                torch.cuda._sleep(10_000_000)
            got = f(*a, stream=s)
            a.clear()
            _scribble(gpu)
            torch.cuda.current_stream().wait_stream(s)
            assert np.array_equal(bits(got), want[n]), (n, strided)
    torch.cuda.synchronize()
    pool.close()


# ------------------------------------------------------------------ a pool's refills and its calls
def _pool(gpu, kind, T, seed):
    """(layer, pool, its blobs on the device, inputs of T tokens): every expert resident, or the first three of
    six, which the routing keeps to."""
    import torch
    lay = make_layer(SWIGLU, seed=seed, expert_std=0.05)
    n = SWIGLU.n_experts if kind == "resident" else 3
    store = HostStore()
    store.add_layer(0, lay.experts)
    pool = ExpertPool(0, lay.spec, n).build()
    for e in range(n):
        pool.touch([e], [0])
        pool.admit(e, store.region(0, e))
    pool.g2s_device(torch.cuda.current_stream().cuda_stream)
    x, idx, w, _ = _layer_inputs(lay.spec, lay, gpu, T, seed=seed + T)
    if kind != "resident":
        idx = np.stack([np.arange(T) % 3, (np.arange(T) + 1) % 3], 1).astype(np.int32)
    ins = to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu)
    blobs = [bytes_dev(b, gpu) for b in lay.experts[:n]]
    torch.cuda.synchronize()
    return lay, pool, blobs, ins


def _refill(pool, blobs, shift, copy):
    """Expert e's slot takes the bytes of expert e + shift."""
    for e in range(len(blobs)):
        b = blobs[(e + shift) % len(blobs)]
        L.check(L.load().brx_pool_refill_from_device_async(pool.device.handle, int(pool.g2s[e]), b.data_ptr(), b.numel(),
                                                           copy.cuda_stream))


def _queued(streams, call, slow):
    """call() on each stream, the ones of `slow` behind some milliseconds of other work."""
    import torch
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            if i in slow:
                torch.cuda._sleep(20_000_000)
            got.append(call())
    return got


@pytest.mark.parametrize("kind", ["resident", "bounded"])
@pytest.mark.parametrize("n, slow", [(2, [0]), (3, [1]), (11, [0, 2, 9])])
@pytest.mark.parametrize("T", [2, 80])
def test_calls_on_every_stream_are_waited_for(gpu, kind, n, slow, T):
    """The pool's sync and its refills wait for the calls of every stream, the slowest not the last."""
    import torch
    lay, pool, blobs, ins = _pool(gpu, kind, T, 300 + n)
    spec, copy = lay.spec, torch.cuda.Stream()
    streams = [torch.cuda.Stream() for _ in range(n)]
    old = bits(mx.moe_forward(spec, pool, *ins))
    torch.cuda.synchronize()
    call = lambda: mx.moe_forward(spec, pool, *ins)   # noqa: E731
    got = _queued(streams, call, slow)
    pool.device.sync()
    assert all(s.query() for s in streams)
    got += _queued(streams, call, slow)
    _refill(pool, blobs, 1, copy)
    torch.cuda.synchronize()
    for g in got:
        assert np.array_equal(bits(g), old)
    new = bits(call())
    assert not np.array_equal(new, old)
    _refill(pool, blobs, 0, copy)
    assert np.array_equal(bits(call()), old)
    pool.device.check()
    pool.close()


@pytest.mark.parametrize("n", [2, 10])
@pytest.mark.parametrize("T", [2, 80])
def test_a_refill_is_waited_for_on_every_stream(gpu, n, T):
    """Calls issued behind a queued refill see its bytes, the second stream's as the first's, products and bf16
    forwards too."""
    import torch
    lay, pool, blobs, ins = _pool(gpu, "resident", T, 400 + n)
    spec, copy = lay.spec, torch.cuda.Stream()
    streams = [torch.cuda.Stream() for _ in range(n)]
    plain = torch.cuda.Stream()
    q = mx.quantize(ins[0])
    tok = torch.arange(T, dtype=torch.int32, device=gpu).repeat_interleave(spec.top_k)
    call = lambda: mx.moe_forward(spec, pool, *ins)   # noqa: E731
    rows = lambda: mx.expert_product(spec, pool, q, tok, ins[1].view(-1), "up_proj")   # noqa: E731
    want = []
    for shift in (0, 1, 2):
        _refill(pool, blobs, shift, copy)
        torch.cuda.synchronize()
        want.append((bits(call()), bits(rows()), bits(layer_forward(spec, pool, *ins))))
        torch.cuda.synchronize()
    for shift in (0, 1, 2):
        with torch.cuda.stream(copy):
            torch.cuda._sleep(20_000_000)
        _refill(pool, blobs, shift, copy)
        got = _queued(streams, call if shift else rows, [])
        with torch.cuda.stream(plain):
            p16 = layer_forward(spec, pool, *ins)
        torch.cuda.synchronize()
        for g in got:
            assert np.array_equal(bits(g), want[shift][0 if shift else 1])
        assert np.array_equal(bits(p16), want[shift][2])
    pool.close()


@pytest.mark.parametrize("T", [2, 80])
def test_capture_and_refills(gpu, T):
    """A capture on a stream the pool has not seen, straight after a refill, then one on a stream with calls of its
    own; the pool is not synchronized inside the second, and is after it. Replays against eager calls, around
    refills that the program orders."""
    import torch
    lay, pool, blobs, ins = _pool(gpu, "resident", T, 500)
    spec, copy = lay.spec, torch.cuda.Stream()
    call = lambda: mx.moe_forward(spec, pool, *ins)   # noqa: E731
    _refill(pool, blobs, 1, copy)
    torch.cuda.synchronize()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for s in (torch.cuda.Stream(), side):
        if s is side:
            with torch.cuda.stream(side):
                call()
            pool.device.sync()
            torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(call())
            if s is side:
                with pytest.raises(L.BrxError, match="captured"):
                    pool.device.sync()
        graphs.append(g)
    pool.device.sync()
    for shift in (0, 1, 2, 0):
        _refill(pool, blobs, shift, copy)
        torch.cuda.synchronize()
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        want = bits(call())
        torch.cuda.synchronize()
        for o in outs:
            assert np.array_equal(bits(o), want), shift
    pool.device.check()
    pool.close()


@pytest.mark.parametrize("T", [2, 80])
def test_the_table_and_the_calls_of_other_streams(gpu, T):
    """Residency moves while a call on one stream is still queued: it reads the experts it was issued with. A
    call on a stream other than the upload's, which is still queued, reads the new ones."""
    import torch
    lay = make_layer(SWIGLU, seed=77, expert_std=0.05)
    spec = lay.spec
    _, _, whole, _ = build_gpu_layer(lay, gpu)
    whole.g2s_device(torch.cuda.current_stream().cuda_stream)
    x, _, w, _ = _layer_inputs(spec, lay, gpu, T, seed=12)
    xd, wd = to_dev_bits(x, gpu), dev(w, gpu)
    low = np.stack([np.arange(T) % 3, (np.arange(T) + 1) % 3], 1).astype(np.int32)
    ids = [dev(low, gpu), dev(low + 3, gpu)]
    want = [bits(mx.moe_forward(spec, whole, xd, i, wd)) for i in ids]
    store = HostStore()
    store.add_layer(0, lay.experts)
    pool = ExpertPool(0, spec, 3).build()
    sw = StreamingSwitchGLU(pool, PinnedFetcher(store), activations="mxfp4")
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for step in range(6):
        i = step % 2
        sw.ensure(low + 3 * i)
        with torch.cuda.stream(b):
            torch.cuda._sleep(10_000_000)
            pool.g2s_device(b.cuda_stream)
        with torch.cuda.stream(a):          # (behind the upload)
            if step % 3:
                torch.cuda._sleep(10_000_000)
            one = mx.moe_forward(spec, pool, xd, ids[i], wd)
        sw.ensure(low + 3 * (1 - i))        # (the slots' next experts wait for the call, and so does the table)
        with torch.cuda.stream(b):
            pool.g2s_device(b.cuda_stream)
            two = mx.moe_forward(spec, pool, xd, ids[1 - i], wd)
        torch.cuda.synchronize()
        assert np.array_equal(bits(one), want[i]) and np.array_equal(bits(two), want[1 - i]), step
    pool.device.check()
    pool.close()
    whole.close()


@pytest.mark.parametrize("kind", ["bounded", "host"])
@pytest.mark.parametrize("T", [2, 90])
def test_a_bounded_switch_on_streams_in_turn(gpu, kind, T):
    """Steps of one bounded layer on three streams in turn, some with work ahead of them, each step with a routing of
    its own: the resident layer's bits."""
    import torch
    lay = make_layer(SHARED, seed=92, expert_std=0.05)
    whole, wpool = _switch(lay, gpu, "resident", "mxfp4")
    sw, pool = _switch(lay, gpu, kind, "mxfp4")
    if kind == "host":
        sw._serve.depth = 2        # (the routing of a step two behind is waited for and acted on)
    steps = []
    for k in range(18):
        x, _, w, sg = _layer_inputs(lay.spec, lay, gpu, T, seed=200 + k)
        # three experts a step, other ones each time (a step of more leaves no slot of three to give up)
        idx = ((np.argsort(np.random.default_rng(k).random((T, 3)), 1) + k) % lay.spec.n_experts).astype(np.int32)
        steps.append((to_dev_bits(x, gpu), dev(idx, gpu), dev(w, gpu), dev(sg, gpu)))
    want = [bits(whole.forward_combined(*s)) for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for k, s in enumerate(steps):
        if k % 4 == 1:
            with torch.cuda.stream(streams[k % 3]):
                torch.cuda._sleep(5_000_000)
        got.append(sw.forward_combined(*s, stream=streams[k % 3]))
    torch.cuda.synchronize()
    for k in range(len(steps)):
        assert np.array_equal(bits(got[k]), want[k]), k
    assert pool.evicts > 0
    pool.device.check()
    pool.close()
    wpool.close()

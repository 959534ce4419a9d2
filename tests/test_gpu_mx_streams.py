"""Layers of MXFP4 experts on streams of the caller's."""
import numpy as np
import pytest

from bigrig_amd import formats as F
from bigrig_amd.layer import MoELayer, StreamingSwitchGLU
from bigrig_amd.pool import ExpertPool, HostStore, PinnedFetcher
from tests.gpu_util import bits, to_dev_bits
from tests.test_gpu_mx import SHARED, _layer_inputs, dev
from tests.gpu_util import build_gpu_layer
from tests.helpers import make_layer

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

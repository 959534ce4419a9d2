"""The operators together, as they are used: a whole expert block and its gradients against fp64, sorted rows through the
library's own experts, norms around its blocks."""
import pytest
import torch

from tests.block_util import close, rand, routing
from tests.gpu_util import build_gpu_layer, to_dev_bits
from tests.helpers import make_layer, make_x, small

pytestmark = pytest.mark.gpu
B, S = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from bigrig_amd import dispatch, grouped, lib, norm
    lib.init(0)
    return dispatch, grouped, norm


def expert_block(ops, x, weights, E, k, idx):
    """The residual stream behind a block of bf16 experts, by the operators."""
    D, G, M = ops
    pre, router, up, down, post, nxt = weights
    h = M.enter(x, pre)
    logits = h.float() @ router.float().t()
    w = torch.softmax(logits.gather(1, idx.long()), -1)
    plan = D.plan(idx, E)
    gu = G.product(D.dispatch(h, plan), up, plan.offsets)
    a, b = gu.float().chunk(2, -1)
    y = G.product((torch.nn.functional.silu(a) * b).to(h.dtype), down, plan.offsets)
    return M.leave(D.combine(y, plan, w), x, post, None, 1.0, nxt)


def expert_block64(x, weights, E, k, idx):
    """The same from the definitions, in the type of its inputs, token by token and expert by expert."""
    pre, router, up, down, post, nxt = weights

    def n(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w

    h = n(x, pre)
    w = torch.softmax((h @ router.t()).gather(1, idx.long()), -1)
    out = torch.zeros_like(x)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            a, b = (h[t] @ up[e].t()).chunk(2, -1)
            out = out.index_add(0, t, w[t, j][:, None] * ((a / (1 + torch.exp(-a)) * b) @ down[e].t()))
    new = x + n(out, post)
    return new, n(new, nxt)


@pytest.mark.parametrize("T,H,I,E,k", [(1, 64, 32, 4, 2), (50, 128, 72, 8, 3), (200, 264, 136, 6, 2)])
def test_a_block_and_its_gradients(ops, T, H, I, E, k):
    idx = routing(T, k, E, T)
    near = lambda shape, seed: (rand(shape, S, seed) * 0.1 + 1.0).to(B)
    weights = [near((H,), 1), rand((E, H), B, 2, scale=0.1), rand((E, 2 * I, H), B, 3, scale=0.1),
               rand((E, H, I), B, 4, scale=0.1), near((H,), 5), near((H,), 6)]
    x = rand((T, H), B, 7)
    leaves = [t.requires_grad_() for t in (x, *weights)]
    outs = expert_block(ops, x, weights, E, k, idx)
    d = [rand((T, H), B, 8), rand((T, H), B, 9)]
    got = [*outs, *torch.autograd.grad(outs, leaves, d)]
    l64 = [t.detach().cpu().double().requires_grad_() for t in leaves]
    o64 = expert_block64(l64[0], l64[1:], E, k, idx.cpu())
    want = [*o64, *torch.autograd.grad(o64, l64, [t.cpu().double() for t in d])]
    # Every tensor on the way (h, gate and up, the activation, y, the sum, new, and as many gradients) is rounded to bf16,
    # each off by at most 2^-8 of its size in every element; a chain of 12 such roundings, each passed on by products that
    # keep relative sizes of whole tensors within a few, is off by 12 x 2^-8 = 4.7e-2 of a tensor's norm at most.
    for i, (a, b) in enumerate(zip(got, want)):
        a = a.detach().cpu().double()
        err = (a - b).norm() / b.norm()
        assert err < 12 * 2.0 ** -8, (i, float(err))


def test_a_captured_block_step(ops):
    T, H, I, E, k = 64, 128, 72, 8, 3
    near = lambda shape, seed: (rand(shape, S, seed) * 0.1 + 1.0).to(B)
    weights = [near((H,), 1), rand((E, H), B, 2, scale=0.1), rand((E, 2 * I, H), B, 3, scale=0.1),
               rand((E, H, I), B, 4, scale=0.1), near((H,), 5), near((H,), 6)]
    x, idx = rand((T, H), B, 7), routing(T, k, E, 1)
    d = [rand((T, H), B, 8), rand((T, H), B, 9)]

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, *weights)]
        outs = expert_block(ops, leaves[0], leaves[1:], E, k, idx)
        return (*outs, *torch.autograd.grad(outs, leaves, d))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        x.copy_(rand((T, H), B, 20 + i))
        idx.copy_(routing(T, k, E, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


def test_blocks_on_two_streams_at_once(ops):
    # calls share nothing: steps of two blocks, queued in turn on two streams with no wait between them
    E, k = 8, 3
    near = lambda shape, seed: (rand(shape, S, seed) * 0.1 + 1.0).to(B)
    jobs = []
    for T, H, I, seed in ((3000, 256, 136, 0), (40, 128, 72, 50)):
        weights = [near((H,), seed + 1), rand((E, H), B, seed + 2, scale=0.1), rand((E, 2 * I, H), B, seed + 3, scale=0.1),
                   rand((E, H, I), B, seed + 4, scale=0.1), near((H,), seed + 5), near((H,), seed + 6)]
        jobs.append((weights, rand((T, H), B, seed + 7), routing(T, k, E, seed), [rand((T, H), B, seed + 8 + i) for i in range(2)]))

    def step(job):
        weights, x, idx, d = job
        leaves = [t.detach().requires_grad_() for t in (x, *weights)]
        outs = expert_block(ops, leaves[0], leaves[1:], E, k, idx)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, d)]

    want = [step(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i])), i


def test_the_largest_calls(ops):
    # 2^23 pairs, rows and tokens of small whole numbers, which every type and sum holds exactly
    D, G, M = ops
    T, k, E, H = 1 << 20, 8, 512, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    idx = torch.randint(-1, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randint(-2, 3, (T, H), generator=g, device="cuda").to(B).requires_grad_()
    weight = torch.randint(0, 2, (E, H, H), generator=g, device="cuda").to(B).requires_grad_()
    plan = D.plan(idx, E)
    flat = idx.reshape(-1)
    kept = flat >= 0
    by = torch.where(kept, flat, E).long().argsort(stable=True)
    n = int(kept.sum())
    assert torch.equal(plan.order[:n].long(), by[:n]) and (plan.order[n:] == -1).all()
    assert torch.equal(plan.offsets[1:].long(), torch.bincount(flat[kept].long(), minlength=E).cumsum(0))
    rows = D.dispatch(x, plan)
    assert torch.equal(rows[:n], x[by[:n] // k]) and not rows[n:].any()
    y = G.product(rows, weight, plan.offsets)
    e = flat.long().clamp(min=0).view(T, k)
    want = torch.zeros((T, H), device="cuda")
    for j in range(k):      # (products of tokens' rows one pair at a time, exact)
        for c in range(H):
            want[:, c] += torch.where(idx[:, j] >= 0, (x.float() * weight.float()[:, c][e[:, j]]).sum(-1), 0.0)
    out = D.combine(y, plan)
    assert torch.equal(out, want.to(B))
    dx, dw = torch.autograd.grad(out, (x, weight), torch.ones_like(out))
    hit = torch.where((idx >= 0)[:, :, None], weight.float().sum(1)[e], 0.0).sum(1)
    assert torch.equal(dx, hit.to(B))
    sums = torch.zeros((E + 1, H), device="cuda", dtype=torch.float64)
    sums.index_add_(0, torch.where(kept, flat, E).long(), x.detach().double().repeat_interleave(k, 0))
    # (sums of some 16000 small whole numbers, exact in fp32, rounded once)
    assert torch.equal(dw, sums[:E, None].expand(E, H, H).float().to(B))
    with pytest.raises(ValueError, match="at most"):
        D.plan(torch.zeros((T + 1, k), dtype=torch.int32, device="cuda"), E)

    T = 1 << 23
    r = torch.ones((T, H), dtype=B, device="cuda")
    r[-1], r[12345678 % T] = 4.0, 2.0
    w = torch.ones(H, dtype=S, device="cuda", requires_grad=True)
    new, h = M.leave(r, r, w, next_weight=w)
    assert torch.equal(h, torch.ones_like(h)) and (new[-1] == 5).all() and (new[0] == 2).all() and (new[12345678 % T] == 3).all()
    (dw,) = torch.autograd.grad(h, w, torch.ones_like(h))
    assert torch.isfinite(dw).all()


def test_sorted_rows_through_the_pair_forms(ops):
    # the plan's rows, as pairs of one token each, through the library's own experts: the layer's rows, bit for bit
    from bigrig_amd import layer as ly
    from bigrig_amd.spec import QWEN3_30B_A3B
    D, _, _ = ops
    spec = small(QWEN3_30B_A3B, hidden=256, inter=128, n_experts=16, top_k=4)
    moe, sw, pool, _ = build_gpu_layer(make_layer(spec, seed=3), torch.device("cuda:0"))
    x = to_dev_bits(make_x(40, spec.hidden, seed=4), torch.device("cuda:0"))
    pool.g2s_device(torch.cuda.current_stream().cuda_stream)
    idx, w, _ = moe.route(x)
    plan = D.plan(idx, spec.n_experts)
    rows = D.dispatch(x, plan)
    expert = idx.reshape(-1)[plan.order.long()].contiguous()
    y = torch.empty_like(rows)
    at = torch.arange(rows.shape[0], dtype=torch.int32, device="cuda")
    ly.forward_pairs(spec, pool, rows, at, expert, None, y, ly.path_flag(40, spec.top_k))
    ref = torch.empty((40, spec.top_k, spec.hidden), dtype=B, device="cuda")
    ly.moe_forward(spec, pool, x, idx, y_unreduced=ref)
    assert torch.equal(y, ref.view(-1, spec.hidden)[plan.order.long()])
    out = torch.empty_like(x)
    ly.combine(spec, ref, w, out)
    # the two sums take a token's rows in one order
    close(D.combine(y, plan, w), out.double(), 2.0 ** -8 * out.double().abs() + 1e-30, "combine")
    pool.close()


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("stream_dtype", [B, S])
def test_norms_around_a_layer(ops, T, stream_dtype):
    from bigrig_amd.spec import QWEN3_30B_A3B
    _, _, M = ops
    spec = small(QWEN3_30B_A3B, hidden=256, inter=128, n_experts=16, top_k=4)
    moe, sw, pool, _ = build_gpu_layer(make_layer(spec, seed=5), torch.device("cuda:0"))
    H = spec.hidden
    x = rand((2, T, H), stream_dtype, 6)
    pre, post, gate = (rand((H,), S, 7 + i) * 0.1 + 1.0 for i in range(3))
    h = M.enter(x, pre, dtype=B)
    y = moe(h)
    want = M.leave(y, x, post, gate, 0.5)
    moe.norms = M.BlockNorms(pre, post, gate, 0.5)
    assert torch.equal(moe(x), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = moe(x, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    # no gradient is recorded: the block has none
    assert not moe(x.clone().requires_grad_()).requires_grad
    pool.close()


def test_prefill_with_norms(ops):
    from bigrig_amd.layered import LayerRing, MoEWeights, prefill
    from bigrig_amd.pool import HostStore
    from bigrig_amd.spec import QWEN3_30B_A3B
    _, _, M = ops
    spec = small(QWEN3_30B_A3B, hidden=256, inter=128, n_experts=8, top_k=2)
    n, dev = 4, torch.device("cuda:0")
    lays = [make_layer(spec, seed=10 + i) for i in range(n)]
    store = HostStore()
    for i, lay in enumerate(lays):
        store.add_layer(i, lay.experts)
    built = [build_gpu_layer(lay, dev) for lay in lays]
    H = spec.hidden
    vec = lambda seed: rand((H,), S, seed) * 0.1 + 1.0
    # the third block has no norms, the fourth another eps: neither's input comes from the pass before
    norms = [M.BlockNorms(vec(1), vec(2), vec(3), 0.5), M.BlockNorms(vec(4)), None, M.BlockNorms(vec(5), eps=1e-3)]
    ring = LayerRing(spec)
    layers = [MoEWeights(i, b[0].router_w, b[0].router_bias, norms=norms[i]) for i, b in enumerate(built)]
    chunks = [rand((t, H), B, 30 + t) for t in (20, 7)]
    got = prefill(spec, layers, store, [c.clone() for c in chunks], ring)
    for x, out in zip(chunks, got):
        for (moe, *_), nm in zip(built, norms):
            if nm is None:
                x = moe(x) + x
            else:
                x = M.leave(moe(M.enter(x, nm.pre, nm.eps)), x, nm.post, nm.gate, nm.scale, eps=nm.eps)
        assert torch.equal(out, x)
    torch.cuda.synchronize()
    ring.close()
    for b in built:
        b[2].close()

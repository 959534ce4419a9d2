"""Pairs sorted by expert, rows there and back, on the GPU against a plain fp64 restatement."""
import numpy as np
import pytest
import torch

from tests.block_util import DTYPES, SUM_U, U32, close, rand, routing

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def D():
    from bigrig_amd import dispatch, lib
    lib.init(0)
    return dispatch


def plain_plan(idx, E):
    """(order, position, offsets) with every dropped pair's position -1, on the CPU."""
    e = idx.cpu().numpy().reshape(-1).astype(np.int64)
    n = e.size
    kept = (e >= 0) & (e < E)
    order = np.full(n, -1, np.int64)
    by = np.argsort(np.where(kept, e, E), kind="stable")[:kept.sum()]
    order[:by.size] = by
    position = np.full(n, -1, np.int64)
    position[by] = np.arange(by.size)
    offsets = np.concatenate(([0], np.cumsum(np.bincount(e[kept], minlength=E))))
    return order, position, offsets


def check_plan(D, idx, E):
    p = D.plan(idx, E)
    order, position, offsets = plain_plan(idx, E)
    assert np.array_equal(p.order.cpu().numpy(), order)
    assert np.array_equal(p.offsets.cpu().numpy(), offsets)
    got = p.position.cpu().numpy().reshape(-1)
    assert np.array_equal(np.where(got < 0, -1, got), position)
    # the dropped pairs name the rows behind the last one, each its own
    assert sorted(-1 - got[got < 0]) == list(range(offsets[-1], got.size))
    return p


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 128), (0, 4, 8), (7, 8, 256), (63, 1, 3), (64, 2, 5), (65, 4, 512),
                                   (333, 8, 60), (2048, 8, 128), (2049, 8, 128), (4097, 4, 512), (40000, 2, 17),
                                   (70001, 8, 128), (3, 64, 100), (50, 3, 2), (2000, 8, 512), (129, 8, 512), (128, 8, 511),
                                   (2048, 8, 512)])
@pytest.mark.parametrize("drop", [0.0, 0.4])
def test_plan(D, T, k, E, drop):
    check_plan(D, routing(T, k, E, T + k, drop), E)


def test_plan_of_one_expert_of_none_and_of_ids_outside(D):
    check_plan(D, torch.full((5000, 8), 3, dtype=torch.int32, device="cuda"), 7)
    check_plan(D, torch.full((3000, 8), -1, dtype=torch.int32, device="cuda"), 7)
    check_plan(D, torch.tensor([[7, -2147483648, 2147483647, 6], [0, 8, 512, -1]], dtype=torch.int32, device="cuda"), 7)


def test_plan_of_many_pairs(D):
    # more pairs than the blocks' first size of chunk covers
    check_plan(D, routing(90001, 8, 512, 5, 0.1), 512)


def test_plan_of_a_strided_routing(D):
    idx = routing(100, 8, 32, 3)
    check_plan(D, idx[:, ::2], 32)
    check_plan(D, idx[::3], 32)


SHAPES = [(1, 1, 4, 1), (1, 8, 64, 2048), (5, 2, 3, 7), (9, 8, 32, 8), (33, 6, 60, 1001), (130, 8, 16, 264), (17, 9, 12, 520),
          (3, 64, 128, 65), (70, 4, 8, 4100), (4, 3, 5, 8192), (600, 8, 64, 72)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", SHAPES)
@pytest.mark.parametrize("drop", [0.0, 0.4])
def test_rows_and_gradients(D, dtype, T, k, E, H, drop):
    idx = routing(T, k, E, 1, drop)
    plan = D.plan(idx, E)
    order, position, offsets = plain_plan(idx, E)
    n, kept = T * k, int(offsets[-1])
    pair = torch.from_numpy(order[:kept])
    x = rand((T, H), dtype, 2).requires_grad_()
    rows = D.dispatch(x, plan)
    want = torch.zeros((n, H), dtype=torch.float64)
    want[:kept] = x.detach().cpu().double()[pair // k]
    assert torch.equal(rows.detach().cpu().double(), want)

    dr = rand((n, H), dtype, 3)
    (dx,) = torch.autograd.grad(rows, x, dr)
    d64 = dr.cpu().double()
    ref = torch.zeros((T, H), dtype=torch.float64).index_add_(0, pair // k, d64[:kept])
    mag = torch.zeros((T, H), dtype=torch.float64).index_add_(0, pair // k, d64[:kept].abs())
    close(dx, ref, k * SUM_U * mag, "dx")

    y, w = rand((n, H), dtype, 4).requires_grad_(), rand((T, k), torch.float32, 5).requires_grad_()
    out = D.combine(y, plan, w)
    y64, w64 = y.detach().cpu().double(), w.detach().cpu().double().reshape(-1)
    term = w64[pair, None] * y64[:kept]
    ref = torch.zeros((T, H), dtype=torch.float64).index_add_(0, pair // k, term)
    mag = torch.zeros((T, H), dtype=torch.float64).index_add_(0, pair // k, term.abs())
    close(out, ref, k * SUM_U * mag, "out")
    dout = rand((T, H), dtype, 6)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    o64 = dout.cpu().double()
    ref = torch.zeros((n, H), dtype=torch.float64)
    ref[:kept] = w64[pair, None] * o64[pair // k]
    close(dy, ref, U32 * ref.abs(), "dy")
    ref, mag = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    ref[pair] = (o64[pair // k] * y64[:kept]).sum(-1)
    mag[pair] = (o64[pair // k] * y64[:kept]).abs().sum(-1)
    close(dw, ref.view(T, k), (H * SUM_U * mag).view(T, k), "dw")

    # the sum without weights, and either gradient alone: the same bits
    one = D.combine(y.detach(), plan)
    assert torch.equal(one, D.combine(y.detach(), plan, torch.ones_like(w)))
    y1, w1 = y.detach().requires_grad_(), w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(D.combine(y1, plan, w.detach()), y1, dout)[0], dy)
    assert torch.equal(torch.autograd.grad(D.combine(y.detach(), plan, w1), w1, dout)[0], dw)


def test_gradients_by_differences(D):
    T, k, E, H = 6, 3, 5, 20
    plan = D.plan(routing(T, k, E, 8, 0.3), E)
    y, w = rand((T * k, H), torch.float32, 9).requires_grad_(), rand((T, k), torch.float32, 10).requires_grad_()
    dout = rand((T, H), torch.float32, 11)
    dy, dw = torch.autograd.grad(D.combine(y, plan, w), (y, w), dout)
    # bilinear: a central difference with a step of 1 is exact but for the sums' roundings
    for grad, leaf in ((dy, y), (dw, w)):
        for at in range(0, leaf.numel(), 7):
            step = torch.zeros(leaf.numel(), device="cuda")
            step[at] = 1.0
            step = step.view(leaf.shape)
            up = D.combine(y + step, plan, w) if leaf is y else D.combine(y, plan, w + step)
            dn = D.combine(y - step, plan, w) if leaf is y else D.combine(y, plan, w - step)
            num = ((up.double() - dn.double()) * dout.double()).sum().item() / 2
            size = ((up.double().abs() + dn.double().abs()) * dout.double().abs()).sum().item()
            assert abs(num - grad.reshape(-1)[at].item()) <= (k + H) * SUM_U * size


def test_dropped_rows_may_hold_anything(D):
    T, k, E, H = 40, 4, 8, 96
    idx = routing(T, k, E, 12, 0.5)
    idx[5] = -1                                     # a token without any expert
    plan = D.plan(idx, E)
    kept = int(plan.offsets[-1])
    y, w = rand((T * k, H), torch.bfloat16, 13), rand((T, k), torch.float32, 14)
    ref = D.combine(y, plan, w)
    y2, w2 = y.clone(), w.clone()
    y2[kept:] = float("nan")
    w2[idx < 0] = float("inf")
    assert torch.equal(D.combine(y2, plan, w2), ref)
    assert torch.equal(ref[5], torch.zeros_like(ref[5]))
    y2, w2 = y2.requires_grad_(), w2.requires_grad_()
    dout = rand((T, H), torch.bfloat16, 15)
    dy, dw = torch.autograd.grad(D.combine(y2, plan, w2), (y2, w2), dout)
    assert torch.isfinite(dy.float()).all() and torch.isfinite(dw).all()
    assert not dy[kept:].any() and not dw[idx < 0].any()
    dr = rand((T * k, H), torch.bfloat16, 16)
    dr[kept:] = float("nan")
    x = rand((T, H), torch.bfloat16, 17).requires_grad_()
    (dx,) = torch.autograd.grad(D.dispatch(x, plan), x, dr)
    assert torch.isfinite(dx.float()).all() and not dx[5].any()


def test_nan_and_infinities_stay_where_they_belong(D):
    T, k, E, H = 12, 4, 8, 64
    plan = D.plan(routing(T, k, E, 18), E)
    y = rand((T * k, H), torch.bfloat16, 19)
    r = int(plan.position[3, 1])
    y[r, 7] = float("nan")
    y[int(plan.position[4, 2]), 9] = float("inf")
    out = D.combine(y, plan, torch.ones((T, k), device="cuda"))
    nan = torch.isnan(out)
    assert nan[3, 7] and nan.sum() == 1 and torch.isinf(out[4, 9])


def test_strided_and_misaligned_rows(D):
    T, k, E, H = 50, 4, 16, 136
    idx = routing(T, k, E, 20)
    plan = D.plan(idx, E)
    for dtype in DTYPES:
        big = rand((2 * T, 3 * H + 1), dtype, 21)
        x = big[::2, 5:5 + H]
        assert torch.equal(D.dispatch(x, plan), D.dispatch(x.contiguous(), plan))
        assert torch.equal(D.dispatch(x[:, ::2], plan), D.dispatch(x[:, ::2].contiguous(), plan))
        flat = rand((T * k * H + 3,), dtype, 22)
        y = flat[3:].view(T * k, H)                 # an address that only its type's alignment holds for
        assert torch.equal(D.combine(y, plan), D.combine(y.clone(), plan))
    # gradients that arrive expanded or transposed
    x = rand((T, H), torch.float32, 23).requires_grad_()
    (a,) = torch.autograd.grad(D.dispatch(x, plan).sum(), x)
    assert torch.equal(a, torch.full_like(a, float(k)))
    y, w = rand((T * k, H), torch.float32, 24).requires_grad_(), torch.ones((T, k), device="cuda").requires_grad_()
    out = D.combine(y, plan, w)
    g = rand((H, T), torch.float32, 25).t()
    one = torch.autograd.grad(out, (y, w), g, retain_graph=True)
    two = torch.autograd.grad(out, (y, w), g.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_rows_past_two_to_the_thirty_one_bytes(D):
    # 300000 x 8 rows of 1024 bf16 values: 4.9 GB
    T, k, E, H = 300000, 8, 128, 1024
    idx = torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda")
    plan = D.plan(idx, E)
    x = (torch.arange(T, device="cuda") % 251).to(torch.bfloat16)[:, None].expand(T, H).contiguous()
    rows = D.dispatch(x, plan)
    tok = (plan.order // k).long()
    assert torch.equal(rows[:, 0], x[tok, 0]) and torch.equal(rows[:, -1], x[tok, -1])
    out = D.combine(rows, plan)
    assert torch.equal(out[:, 0].float(), (8 * x[:, 0].float()).to(torch.bfloat16).float())
    assert torch.equal(out[:, -1], out[:, 0])


def test_streams_and_graphs(D):
    T, k, E, H = 300, 8, 64, 520
    idx, w = routing(T, k, E, 26), rand((T, k), torch.float32, 27)
    x = rand((T, H), torch.bfloat16, 28)
    plan = D.plan(idx, E)
    ref = D.combine(D.dispatch(x, plan), plan, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    p2 = D.plan(idx, E, stream=s)
    got = D.combine(D.dispatch(x, p2, stream=s), p2, w, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref) and torch.equal(p2.order, plan.order)

    # gradients of calls given a stream
    gx, gw = x.clone().requires_grad_(), w.clone().requires_grad_()
    d = rand((T, H), torch.bfloat16, 60)
    want = torch.autograd.grad(D.combine(D.dispatch(gx, plan), plan, gw), (gx, gw), d)
    s.wait_stream(torch.cuda.current_stream())
    rows = D.dispatch(gx, plan, stream=s)
    out = D.combine(rows, plan, gw, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (gx, gw), d), want))

    sx, si, sw, sd = x.clone(), idx.clone(), w.clone(), rand((T, H), torch.bfloat16, 29)

    def step():
        px, pw = sx.detach().requires_grad_(), sw.detach().requires_grad_()
        p = D.plan(si, E)
        o = D.combine(D.dispatch(px, p), p, pw)
        return (o, *torch.autograd.grad(o, (px, pw), sd))

    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        sx.copy_(rand((T, H), torch.bfloat16, 30 + i))
        si.copy_(routing(T, k, E, 40 + i, 0.2))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


def test_every_run_gives_the_same_bits(D):
    T, k, E, H = 2000, 8, 64, 264
    idx, w = routing(T, k, E, 50, 0.1), rand((T, k), torch.float32, 51).requires_grad_()
    y, d = rand((T * k, H), torch.bfloat16, 52).requires_grad_(), rand((T, H), torch.bfloat16, 53)
    ref = None
    for _ in range(3):
        p = D.plan(idx, E)
        o = D.combine(y, p, w)
        got = [p.order, p.position, o.detach(), *torch.autograd.grad(o, (y, w), d)]
        ref = ref or got
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_gradient_of_a_gradient_is_refused(D):
    plan = D.plan(routing(4, 2, 3, 1), 3)
    x = rand((4, 8), torch.float32, 1).requires_grad_()
    with pytest.raises(RuntimeError, match="taken once"):
        torch.autograd.grad(D.dispatch(x, plan).sum(), x, create_graph=True)
    y = rand((8, 8), torch.float32, 2).requires_grad_()
    with pytest.raises(RuntimeError, match="taken once"):
        torch.autograd.grad(D.combine(y, plan).sum(), y, create_graph=True)

"""Norms at both ends of a block and their gradients on the GPU against fp64 formulas."""
import itertools

import pytest
import torch

from tests.block_util import SUM_U, U32, close, half, rand, tiny

pytestmark = pytest.mark.gpu
B, F, S = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6
U = SUM_U


@pytest.fixture(scope="module")
def M():
    from bigrig_amd import lib, norm
    lib.init(0)
    return norm


def c64(t):
    return None if t is None else t.detach().cpu().double()


def stat(v, eps=EPS):
    """Reciprocal root mean square of rows, fp64 [T, 1]."""
    return ((v * v).mean(-1, keepdim=True) + eps).rsqrt()


def back(v, s, g):
    n = v * s
    return s * (g - n * (g * n).mean(-1, keepdim=True))


def back_size(v, s, g):
    """Sum of the magnitudes that `back` adds."""
    n = (v * s).abs()
    return s * (g.abs() + n * (g.abs() * n).mean(-1, keepdim=True))


SIZES = [(1, 1), (1, 2880), (3, 7), (5, 8), (2, 65), (33, 512), (19, 520), (9, 1001), (300, 1024), (7, 1032), (40, 2048),
         (11, 2056), (6, 4099), (2, 8192), (1500, 72)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("xd,hd", [(B, B), (F, F), (S, S), (S, B), (S, F)])
def test_enter(M, T, H, xd, hd):
    x = rand((T, H), xd, 1, scale=3.0).requires_grad_()
    for wd in (B, S, None):
        w = None if wd is None else (rand((H,), S, 2) * 0.2 + 1.0).to(wd).requires_grad_()
        h = M.enter(x, w, EPS, hd)
        assert h.dtype == hd
        v, w64 = c64(x), c64(w) if w is not None else torch.ones(H, dtype=torch.float64)
        s = stat(v)
        # H squares summed, a root, two products
        close(h, v * s * w64, (0.5 * H + 8) * U * (v * s * w64).abs(), "h")
        d = rand((T, H), hd, 3)
        got = torch.autograd.grad(h, [x] + ([w] if w is not None else []), d)
        g = c64(d) * w64
        close(got[0], back(v, s, g), (2 * H + 32) * U * back_size(v, s, g), "dx")
        if w is not None:
            t = c64(d) * v * s
            close(got[1], t.sum(0), (T + 0.5 * H + 8) * U * t.abs().sum(0), "dw")


FORMS = [(post, gate, nxt) for post, gate, nxt in itertools.product((0, 1), ("none", "channel", "row", "full"), (0, 1))]


def leave_case(M, T, H, yd, rd, post, gate, nxt, wd, scale=0.5, seed=0):
    y, r = rand((T, H), yd, seed, scale=2.0).requires_grad_(), rand((T, H), rd, seed + 1, scale=3.0).requires_grad_()
    near = lambda shape, k: (rand(shape, S, seed + k) * 0.2 + 1.0).to(wd).requires_grad_()
    wp = near((H,), 2) if post else None
    gt = {"none": None, "channel": (H,), "row": (T, 1), "full": (T, H)}[gate]
    gt = None if gt is None else near(gt, 3)
    wn = near((H,), 4) if nxt else None
    got = M.leave(y, r, wp, gt, scale, wn, EPS)
    new, h = got if nxt else (got, None)
    assert new.dtype == rd and (h is None or h.dtype == yd)
    y64, r64 = c64(y), c64(r)
    sy = stat(y64) if post else torch.ones((T, 1), dtype=torch.float64)
    w64 = c64(wp) if post else torch.ones(H, dtype=torch.float64)
    g64 = c64(gt) if gt is not None else torch.ones((), dtype=torch.float64)
    u = y64 * sy * w64
    add = scale * g64 * u
    close(new, r64 + add, (0.5 * H + 8) * U * add.abs() + U32 * r64.abs(), "new")
    n64 = c64(new)
    d_new, d_h = rand((T, H), rd, seed + 5), rand((T, H), yd, seed + 6)
    D, size = c64(d_new), c64(d_new).abs()
    if nxt:
        sn, wn64 = stat(n64), c64(wn)
        close(h, n64 * sn * wn64, (0.5 * H + 8) * U * (n64 * sn * wn64).abs(), "h")
        q = c64(d_h) * wn64
        D, size = D + back(n64, sn, q), size + back_size(n64, sn, q)
    leaves = [t for t in (y, r, wp, gt, wn) if t is not None]
    grads = list(torch.autograd.grad(got if nxt else [new], leaves, [d_new, d_h] if nxt else [d_new]))
    rel = (2 * H + 32) * U                       # what D, a product of it or a mean of products is off by, relative to `size`
    dy, dr = grads.pop(0), grads.pop(0)
    close(dr, D, rel * size, "dr")
    du, du_size = scale * g64 * D, (scale * g64).abs() * size
    if post:
        close(dy, back(y64, sy, du * w64), 2 * rel * back_size(y64, sy, du_size * w64.abs()), "dy")
        close(grads.pop(0), (du * y64 * sy).sum(0), (2 * rel + T * U) * (du_size * (y64 * sy).abs()).sum(0), "dpost")
    else:
        close(dy, du, 2 * rel * du_size, "dy")
    if gt is not None:
        dg, dg_size = scale * u * D, abs(scale) * u.abs() * size
        dims = {"channel": 0, "row": 1, "full": None}[gate]
        if dims is not None:
            dg, dg_size = dg.sum(dims, keepdim=gate == "row"), dg_size.sum(dims, keepdim=gate == "row")
        close(grads.pop(0), dg, (2 * rel + (T + H) * U) * dg_size, "dgate")
    if nxt:
        t = c64(d_h) * n64 * sn
        close(grads.pop(0), t.sum(0), (T + 0.5 * H + 8) * U * t.abs().sum(0), "dnext")
        # one call gives the bits of the two
        assert torch.equal(new, M.leave(y, r, wp, gt, scale, eps=EPS))
        assert torch.equal(h, M.enter(new.detach(), wn, EPS, yd))
    # without gradients: the same bits
    with torch.no_grad():
        again = M.leave(y, r, wp, gt, scale, wn, EPS)
    assert all(torch.equal(a, b) for a, b in zip(again if nxt else [again], got if nxt else [got]))


@pytest.mark.parametrize("post,gate,nxt", FORMS)
@pytest.mark.parametrize("T,H", [(1, 2880), (37, 520), (5, 1001), (21, 2048), (3, 7)])
def test_leave_forms(M, post, gate, nxt, T, H):
    leave_case(M, T, H, B, B, post, gate, nxt, B)


@pytest.mark.parametrize("yd,rd,wd", [(F, F, F), (S, S, S), (B, S, B), (F, S, S), (B, B, S), (B, S, F)])
@pytest.mark.parametrize("gate", ["channel", "row", "full"])
def test_leave_types(M, yd, rd, wd, gate):
    leave_case(M, 23, 264, yd, rd, 1, gate, 1, wd)
    leave_case(M, 9, 1500, yd, rd, 1, gate, 1, wd, scale=-1.25)


@pytest.mark.parametrize("T,H", SIZES)
def test_leave_sizes(M, T, H):
    leave_case(M, T, H, B, S, 1, "channel", 1, B)


def test_only_what_is_asked_for(M):
    T, H = 30, 264
    y, r, w, g, n = rand((T, H), B, 1), rand((T, H), B, 2), rand((H,), B, 3), rand((H,), B, 4), rand((H,), B, 5)
    d = [rand((T, H), B, 6), rand((T, H), B, 7)]
    whole = [t.clone().requires_grad_() for t in (y, r, w, g, n)]
    ref = torch.autograd.grad(M.leave(*whole[:4], 0.5, whole[4]), whole, d)
    for i in range(5):
        ts = [t.clone() for t in (y, r, w, g, n)]
        ts[i].requires_grad_()
        out = M.leave(*ts[:4], 0.5, ts[4])
        (got,) = torch.autograd.grad(out, ts[i], d)
        assert torch.equal(got, ref[i]), i
    # one of the two results unused
    new, h = M.leave(*whole[:4], 0.5, whole[4])
    a = torch.autograd.grad(new, whole[:4], d[0])
    b = torch.autograd.grad(M.leave(*whole[:4], 0.5), whole[:4], d[0])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    new, h = M.leave(*whole[:4], 0.5, whole[4])
    a = torch.autograd.grad(h, whole, d[1])
    new, h = M.leave(*whole[:4], 0.5, whole[4])
    b = torch.autograd.grad([new, h], whole, [torch.zeros_like(new), d[1]])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradients_by_differences(M):
    T, H = 3, 12
    ts = [rand((T, H), S, 1), rand((T, H), S, 2), rand((H,), S, 3) + 2, rand((T, 1), S, 4), rand((H,), S, 5) + 2]
    d = [rand((T, H), S, 6), rand((T, H), S, 7)]
    leaves = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(M.leave(*leaves[:4], 0.7, leaves[4], eps=1e-3), leaves, d)

    def value(*v):
        new, h = M.leave(*v[:4], 0.7, v[4], eps=1e-3)
        return (new.double() * d[0].double()).sum().item() + (h.double() * d[1].double()).sum().item()

    # a step of 2^-6: the third derivative's share is of order step^2 (values and weights of a few units: below 100 step^2),
    # the roundings' of order U32 * sum / step
    step = 2.0 ** -6
    noise = 40 * T * H * U32 * 30 / step
    for i, leaf in enumerate(ts):
        for at in range(0, leaf.numel(), 5):
            e = torch.zeros(leaf.numel(), device="cuda")
            e[at] = step
            e = e.view(leaf.shape)
            up = value(*[t + e if j == i else t for j, t in enumerate(ts)])
            dn = value(*[t - e if j == i else t for j, t in enumerate(ts)])
            assert abs((up - dn) / (2 * step) - grads[i].reshape(-1)[at].item()) <= 100 * step * step + noise, (i, at)


def test_rows_of_zero_and_of_extremes(M):
    H = 520
    x = torch.zeros((6, H), dtype=B, device="cuda")
    x[1] = 1e-30
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    x[4] = 60000.0
    x[5, 0] = 1.0
    h = M.enter(x, None, EPS)
    assert not h[0].any() and torch.isfinite(h[1].float()).all() and torch.isnan(h[2]).all()
    assert torch.isnan(h[3, 4]) and not h[3, :4].any()      # inf * 0, and finite values over an infinite root
    close(h[4], torch.ones(H, dtype=torch.float64), (0.5 * H + 8) * U, "large")
    xr = x[[0, 1, 4, 5]].clone().requires_grad_()
    (g,) = torch.autograd.grad(M.enter(xr, None, EPS), xr, torch.ones_like(xr))
    assert torch.isfinite(g.float()).all()
    f = torch.full((2, 96), 65504.0, dtype=F, device="cuda")
    close(M.enter(f, None, EPS), torch.ones((2, 96), dtype=torch.float64), (0.5 * 96 + 8) * U, "fp16")


def test_strides_and_shapes(M):
    for dtype in (B, F, S):
        big = rand((2, 40, 3, 201), dtype, 1)
        for x in (big[0, :, 0, 5:134], big[:, ::2, 1, :129], big[:, :, :, 3:132], big.transpose(1, 3)[0, :150, 0, :40],
                  big[0, 0, 0, 1:130]):
            H = x.shape[-1]
            w = rand((H,), dtype, 2)
            assert torch.equal(M.enter(x, w), M.enter(x.contiguous(), w))
            y = rand(x.shape, dtype, 3)
            one = M.leave(x, y, w, None, 1.0, w)
            two = M.leave(x.contiguous(), y, w, None, 1.0, w)
            assert one[0].shape == x.shape and all(torch.equal(a, b) for a, b in zip(one, two))
            assert torch.equal(M.leave(y, x), M.leave(y, x.contiguous()))
            g = rand((*x.shape[:-1], 1), dtype, 4)
            if x.dim() > 1:
                assert torch.equal(M.leave(x, y, None, g), M.leave(x, y, None, g.expand(x.shape)))
    # gradients that arrive expanded or transposed, of inputs that are views
    x = rand((3, 50, 264), B, 5)[:, ::2].requires_grad_()
    h = M.enter(x, None)
    a = torch.autograd.grad(h, x, torch.ones((1, 1, 1), dtype=B, device="cuda").expand(h.shape), retain_graph=True)[0]
    b = torch.autograd.grad(h, x, torch.ones_like(h))[0]
    assert torch.equal(a, b)


def test_no_rows(M):
    H = 72
    y, r = (torch.empty((0, H), dtype=B, device="cuda").requires_grad_() for _ in range(2))
    w, g, n = (rand((H,), B, i).requires_grad_() for i in range(3))
    new, h = M.leave(y, r, w, g, 1.0, n)
    assert new.shape == h.shape == (0, H)
    grads = torch.autograd.grad([new, h], (y, r, w, g, n), [torch.empty_like(new), torch.empty_like(h)])
    assert grads[0].shape == (0, H) and not any(t.any() for t in grads[2:])
    assert M.enter(y.detach().view(2, 0, H), w).shape == (2, 0, H)


def test_many_rows(M):
    # several rows a block in the column sums, and rows past 2^31 bytes
    leave_case(M, 9000, 264, B, B, 1, "channel", 1, S)
    T, H = 600000, 2048
    x = torch.ones((T, H), dtype=B, device="cuda")
    x[-1] = 3.0
    h = M.enter(x, None)
    assert (h[-1] == 1).all() and (h[0] == 1).all() and (M.leave(x, x)[-1] == 6).all()


def test_streams_and_graphs(M):
    T, H = 200, 520
    ts = [rand((T, H), B, 1), rand((T, H), S, 2), rand((H,), B, 3), rand((H,), B, 4), rand((H,), B, 5)]
    d = [rand((T, H), S, 6), rand((T, H), B, 7)]

    def step():
        v = [t.detach().requires_grad_() for t in ts]
        out = M.leave(*v[:4], 0.5, v[4])
        return (*out, *torch.autograd.grad(out, v, d))

    ref = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = M.leave(*ts[:4], 0.5, ts[4], stream=s)
    h = M.enter(ts[0], ts[2], stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]) and torch.equal(h, M.enter(ts[0], ts[2]))
    v = [t.clone().requires_grad_() for t in ts]
    s.wait_stream(torch.cuda.current_stream())
    got = M.leave(*v[:4], 0.5, v[4], stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(got, v, d), ref[2:]))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        for j, t in enumerate(ts):
            t.copy_(rand(t.shape, t.dtype, 10 * i + j))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


def test_gradient_of_a_gradient_is_refused(M):
    x, r = rand((4, 8), S, 1).requires_grad_(), rand((4, 8), S, 2)
    for out in (M.enter(x), M.leave(x, r)):
        with pytest.raises(RuntimeError, match="taken once"):
            torch.autograd.grad(out.sum(), x, create_graph=True)

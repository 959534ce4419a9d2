"""Grouped products and their gradients on the GPU against fp64 products."""
import pytest
import torch

from tests.block_util import SUM_U, close, rand

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def G():
    from bigrig_amd import grouped, lib
    lib.init(0)
    return grouped


def offsets_of(counts):
    t = torch.tensor([0] + list(counts), dtype=torch.int64).cumsum(0)
    return t.int().cuda(), t.tolist()


def reference(rows, weight, at, bias, dout):
    """(out, its magnitude, and the same of drows, dweight, dbias), fp64 on the CPU."""
    x, w, d = rows.detach().cpu().double(), weight.detach().cpu().double(), dout.cpu().double()
    P, E = x.shape[0], w.shape[0]
    N, K = w.shape[1:]
    r = {n: torch.zeros(s, dtype=torch.float64) for n, s in
         (("out", (P, N)), ("out_m", (P, N)), ("drows", (P, K)), ("drows_m", (P, K)), ("dw", (E, N, K)), ("dw_m", (E, N, K)),
          ("db", (E, N)), ("db_m", (E, N)))}
    for e in range(E):
        s = slice(at[e], at[e + 1])
        r["out"][s], r["out_m"][s] = x[s] @ w[e].T, x[s].abs() @ w[e].T.abs()
        if bias is not None:
            b = bias.detach().cpu().double()[e]
            r["out"][s] += b
            r["out_m"][s] += b.abs()
        r["drows"][s], r["drows_m"][s] = d[s] @ w[e], d[s].abs() @ w[e].abs()
        r["dw"][e], r["dw_m"][e] = d[s].T @ x[s], d[s].T.abs() @ x[s].abs()
        r["db"][e], r["db_m"][e] = d[s].sum(0), d[s].abs().sum(0)
    return r


def check(G, counts, N, K, dtype, bias=True, behind=0, seed=0):
    offsets, at = offsets_of(counts)
    E, P = len(counts), at[-1] + behind
    rows = rand((P, K), dtype, seed).requires_grad_()
    weight = rand((E, N, K), dtype, seed + 1, scale=0.1).requires_grad_()
    b = rand((E, N), dtype, seed + 2).requires_grad_() if bias else None
    dout = rand((P, N), dtype, seed + 3)
    if behind:      # what lies behind the last run enters nothing
        with torch.no_grad():
            rows[at[-1]:] = float("nan")
            dout[at[-1]:] = float("inf")
    out = G.product(rows, weight, offsets, b)
    ref = reference(rows, weight, at, b, dout)
    close(out, ref["out"], (K + 1) * SUM_U * ref["out_m"], "out")
    grads = torch.autograd.grad(out, [rows, weight] + ([b] if bias else []), dout)
    close(grads[0], ref["drows"], N * SUM_U * ref["drows_m"], "drows")
    most = max(counts) if counts else 0
    close(grads[1], ref["dw"], most * SUM_U * ref["dw_m"], "dweight")
    if bias:
        close(grads[2], ref["db"], most * SUM_U * ref["db_m"], "dbias")


COUNTS = {"one": [1], "none": [0, 0, 0], "single": [1] * 8, "ragged": [0, 3, 129, 0, 64, 1, 128, 17, 0],
          "long": [700, 0, 33], "tail": [127, 255, 31, 65]}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("N,K", [(8, 8), (64, 64), (72, 200), (256, 136), (136, 328), (520, 72)])
def test_products_and_gradients(G, dtype, name, N, K):
    check(G, COUNTS[name], N, K, dtype, bias=(N + K) % 3 != 0, seed=N + K)


@pytest.mark.parametrize("behind", [1, 70, 300])
def test_rows_behind_the_last_run_are_zero_and_enter_nothing(G, behind):
    check(G, [5, 0, 140, 9], 96, 104, torch.bfloat16, behind=behind)


@pytest.mark.parametrize("E,per", [(512, 3), (257, 1), (128, 9), (64, 0)])
def test_many_experts(G, E, per):
    counts = [(i * 7 + per) % (2 * per + 1) for i in range(E)]
    check(G, counts, 64, 72, torch.bfloat16, bias=False)


def test_wide(G):
    check(G, [40, 3], 8192, 264, torch.bfloat16, bias=False)
    check(G, [40, 3], 264, 8192, torch.float16, bias=True)


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, True), (torch.float16, False)])
@pytest.mark.parametrize("N,K", [(4104, 72), (72, 4104)])
def test_enough_rows_for_the_persistent_tiles(G, dtype, bias, N, K):
    # 17 whole tiles of 256 rows by 17 of 256 columns (forward, or the rows' gradient): tiles of 1 to 4 fragments a wave, runs
    # that end in each, empty ones, rows behind the last; sums of one stage, of several, and ending inside one
    counts = [0, 1, 64, 65, 128, 129, 192, 193, 256, 257, 0, 700, 1500, 33, 1000, 0]
    check(G, counts, N, K, dtype, bias=bias, behind=300)


@pytest.mark.parametrize("dtype,bias", [(torch.float16, True), (torch.bfloat16, False)])
def test_enough_rows_for_whole_tiles_of_128(G, dtype, bias):
    # (23 + 10) row tiles by 9 column tiles of 128 both ways, more than the CUs; 11 by 5 of 256, fewer
    check(G, [0, 700, 1, 128, 129, 900, 0, 1000, 127], 1032, 1096, dtype, bias=bias, behind=40)


def test_persistent_tiles_of_more_than_the_cus(G):
    # every block takes several tiles, short sums among long ones
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 300, (200,), generator=g).tolist()
    check(G, counts, 1032, 200, torch.bfloat16, bias=True, behind=5)
    check(G, counts, 1032, 56, torch.float16, bias=False)


def test_persistent_tiles_keep_a_nan_in_its_row(G):
    N, K = 4104, 72
    offsets, at = offsets_of([3, 500, 130, 0, 4000])
    rows, w = rand((at[-1], K), torch.bfloat16, 1), rand((5, N, K), torch.bfloat16, 2)
    ref = G.product(rows, w, offsets)
    bad = rows.clone()
    bad[[2, 3, 502, 700]] = float("nan")
    out = G.product(bad, w, offsets)
    keep = torch.ones(at[-1], dtype=torch.bool, device="cuda")
    keep[[2, 3, 502, 700]] = False
    assert torch.isnan(out[~keep]).all() and torch.equal(out[keep], ref[keep])
    wr = w.clone().requires_grad_()
    d = rand((at[-1], N), torch.bfloat16, 3)
    bad = rows.clone()
    bad[2] = float("nan")
    (g,) = torch.autograd.grad(G.product(bad, wr, offsets), wr, d)
    assert torch.isnan(g[0]).all() and torch.isfinite(g[1:].float()).all() and not g[3].any()


def test_thin_and_square_tiles_agree_with_the_persistent_ones_row_by_row(G):
    # a row's value does not depend on how many others there are, up to the order of its fp32 sum
    N, K = 4104, 264
    w = rand((4, N, K), torch.bfloat16, 1, scale=0.1)
    rows = rand((4800, K), torch.bfloat16, 2)
    full = G.product(rows, w, offsets_of([1200] * 4)[0])
    for take in (1, 5, 8, 40, 300):
        pick = torch.cat([torch.arange(e * 1200, e * 1200 + take) for e in range(4)]).cuda()
        part = G.product(rows[pick], w, offsets_of([take] * 4)[0])
        m = rows[pick].double().cpu().abs() @ torch.ones(K, dtype=torch.float64)
        # (weights are below 0.6 in size: 0.1 times normal values below 6; two fp32 sums and the other's rounding)
        close(part, full[pick].double().cpu(), 2 * K * SUM_U * 0.6 * m[:, None] + 2.0 ** -8 * full[pick].double().cpu().abs(),
              f"{take}")


def test_a_long_run_beside_short_ones(G):
    check(G, [1, 3000, 1], 136, 72, torch.bfloat16)


def test_no_rows(G):
    offsets, _ = offsets_of([0, 0])
    rows = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda").requires_grad_()
    w = rand((2, 32, 64), torch.bfloat16, 1).requires_grad_()
    b = rand((2, 32), torch.bfloat16, 2).requires_grad_()
    out = G.product(rows, w, offsets, b)
    assert out.shape == (0, 32)
    grads = torch.autograd.grad(out, (rows, w, b), torch.empty_like(out))
    assert grads[0].shape == (0, 64) and not grads[1].any() and not grads[2].any()


def test_weights_that_are_parts_of_others(G):
    E, N, K = 4, 96, 72
    offsets, at = offsets_of([7, 0, 150, 3])
    rows, dout = rand((160, K), torch.bfloat16, 1), rand((160, N), torch.bfloat16, 2)
    big = rand((E, 3 * N, 2 * K), torch.bfloat16, 3)
    for w in (big[:, N:2 * N, 8:8 + K], big[:, ::2, :K][:, :N], big[:1, :N, :K].expand(E, N, K), big.flip(0)[::1, :N, :K]):
        a, c = w.detach().requires_grad_(), w.contiguous().requires_grad_()
        rr = rows.clone().requires_grad_()
        o1, o2 = G.product(rr, a, offsets), G.product(rr, c, offsets)
        assert torch.equal(o1, o2)
        g1, g2 = torch.autograd.grad(o1, (rr, a), dout), torch.autograd.grad(o2, (rr, c), dout)
        assert torch.equal(g1[0], g2[0]) and torch.equal(g1[1], g2[1])
    # matrices that experts share: their gradients come summed
    one = rand((1, N, K), torch.float16, 4).requires_grad_()
    r16, d16 = rows.half(), dout.half()
    (g,) = torch.autograd.grad(G.product(r16, one.expand(E, N, K), offsets), one, d16)
    x, d = r16.cpu().double(), d16.cpu().double()
    n = at[-1]
    # the experts' gradients are rounded each, and so are their partial sums
    m = d[:n].abs().T @ x[:n].abs()
    close(g[0], d[:n].T @ x[:n], (2 * E * 2.0 ** -11 + n * SUM_U) * m, "shared")


def test_strided_and_misaligned_rows_and_gradients(G):
    E, N, K = 3, 64, 40
    offsets, at = offsets_of([5, 60, 9])
    big = rand((80, 200), torch.bfloat16, 1)
    w = rand((E, N, K), torch.bfloat16, 2).requires_grad_()
    for rows in (big[:74, 3:3 + K], big[1:75, :K], big.t()[:K].t()[:74]):
        assert torch.equal(G.product(rows, w, offsets), G.product(rows.contiguous().clone(), w, offsets))
    rows = rand((74, K), torch.bfloat16, 3).requires_grad_()
    out = G.product(rows, w, offsets)
    for d in (torch.ones((1, 1), dtype=torch.bfloat16, device="cuda").expand(74, N), rand((N, 74), torch.bfloat16, 4).t(),
              rand((74 * N + 1,), torch.bfloat16, 5)[1:].view(74, N)):
        a = torch.autograd.grad(out, (rows, w), d, retain_graph=True)
        b = torch.autograd.grad(out, (rows, w), d.clone().contiguous(), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_nan_stays_in_its_row(G):
    # the widths end inside a stage and inside a tile, the runs next to one another
    offsets, _ = offsets_of([3, 4, 130])
    rows, w = rand((137, 72), torch.bfloat16, 1), rand((3, 136, 72), torch.bfloat16, 2)
    ref = G.product(rows, w, offsets)
    bad = rows.clone()
    bad[3] = float("nan")
    out = G.product(bad, w, offsets)
    assert torch.isnan(out[3]).all()
    keep = torch.arange(137, device="cuda") != 3
    assert torch.equal(out[keep], ref[keep])
    # another expert's matrix of NaN reaches its own rows only, and no other expert's gradient
    wb = w.clone()
    wb[1] = float("nan")
    out = G.product(rows, wb, offsets)
    assert torch.equal(out[:3], ref[:3]) and torch.equal(out[7:], ref[7:]) and torch.isnan(out[3:7]).all()
    wr = w.clone().requires_grad_()
    d = rand((137, 136), torch.bfloat16, 3)
    (g,) = torch.autograd.grad(G.product(bad, wr, offsets), wr, d)
    assert torch.isfinite(g[0].float()).all() and torch.isfinite(g[2].float()).all() and torch.isnan(g[1]).all()


def test_offsets_out_of_order_or_range_touch_nothing_else(G):
    E, N, K, P = 4, 40, 72, 50
    rows, w = rand((P, K), torch.bfloat16, 1).requires_grad_(), rand((E, N, K), torch.bfloat16, 2).requires_grad_()
    for o in ([0, 60, -5, 100, 1 << 30], [5, 10, 10, 20, 20], [0, 30, 10, 40, 50], [-(1 << 31), 0, 0, 0, 0]):
        off = torch.tensor(o, dtype=torch.int32, device="cuda")
        out = G.product(rows, w, off)
        torch.autograd.grad(out, (rows, w), torch.ones_like(out))
    torch.cuda.synchronize()


def test_matrix_gradients_larger_than_the_caches(G):
    E, N, K = 65, 2056, 1088         # 291 MB of whole lines, tiles of 8 rows at their end
    counts = [0 if e % 9 == 4 else e % 7 * 13 + 1 for e in range(E)]
    offsets, at = offsets_of(counts)
    rows, dout = rand((at[-1], K), torch.bfloat16, 1), rand((at[-1], N), torch.bfloat16, 2)
    w = torch.zeros((E, N, K), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    for _ in range(2):
        (dw,) = torch.autograd.grad(G.product(rows, w, offsets), w, dout)
        for e in range(E):
            if not counts[e]:
                assert not dw[e].any(), e
            elif e % 8 == 0 or e == E - 1:
                x, d = (t[at[e]:at[e + 1]].cpu().double() for t in (rows, dout))
                close(dw[e], d.T @ x, counts[e] * SUM_U * (d.abs().T @ x.abs()), f"dweight of {e}")


def test_rows_past_two_to_the_thirty_one_bytes(G):
    P, K, N = 600000, 2048, 8        # 2.5 GB of rows, one expert
    offsets, _ = offsets_of([10, P - 10])
    rows = torch.zeros((P, K), dtype=torch.bfloat16, device="cuda")
    rows[-1] = 1.0
    rows[5] = 2.0
    w = torch.ones((2, N, K), dtype=torch.bfloat16, device="cuda").requires_grad_()
    out = G.product(rows, w, offsets)
    assert (out[-1] == 2048).all() and (out[5] == 4096).all() and not out[10:-1].any()
    d = torch.zeros_like(out)
    d[-1] = 3.0
    (g,) = torch.autograd.grad(out, w, d)
    assert (g[1] == 3).all() and not g[0].any()


def test_streams_and_graphs(G):
    E, N, K, P = 6, 136, 200, 300
    counts = [[10, 0, 200, 30, 60, 0], [300, 0, 0, 0, 0, 0], [0, 50, 50, 50, 50, 100], [1, 2, 3, 4, 5, 6]]
    offsets, _ = offsets_of(counts[0])
    rows, w, b = rand((P, K), torch.bfloat16, 1), rand((E, N, K), torch.bfloat16, 2), rand((E, N), torch.bfloat16, 3)
    d = rand((P, N), torch.bfloat16, 4)

    def step():
        lr, lw, lb = (t.detach().requires_grad_() for t in (rows, w, b))
        out = G.product(lr, lw, offsets, lb)
        return (out, *torch.autograd.grad(out, (lr, lw, lb), d))

    ref = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = G.product(rows, w, offsets, b, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref[0])
    lr, lw, lb = (t.clone().requires_grad_() for t in (rows, w, b))
    s.wait_stream(torch.cuda.current_stream())
    out = G.product(lr, lw, offsets, lb, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(out, (lr, lw, lb), d), ref[1:]))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        offsets.copy_(offsets_of(counts[i])[0])
        rows.copy_(rand((P, K), torch.bfloat16, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, step()):
            assert torch.equal(a, c), i


def test_gradient_by_differences(G):
    # fp16 inputs that are small whole numbers: sums and differences are exact
    E, N, K, P = 2, 8, 16, 12
    offsets, _ = offsets_of([5, 7])
    whole = lambda shape, seed: rand(shape, torch.float32, seed, scale=2.0).round().half()
    rows, w, d = whole((P, K), 1).requires_grad_(), whole((E, N, K), 2).requires_grad_(), whole((P, N), 3)
    out = G.product(rows, w, offsets)
    gr, gw = torch.autograd.grad(out, (rows, w), d)
    for leaf, grad in ((rows, gr), (w, gw)):
        for at in range(0, leaf.numel(), 11):
            step = torch.zeros(leaf.numel(), dtype=torch.float16, device="cuda")
            step[at] = 1.0
            step = step.view(leaf.shape)
            up = G.product(rows + step, w, offsets) if leaf is rows else G.product(rows, w + step, offsets)
            num = ((up.double() - out.double()) * d.double()).sum().item()
            assert num == grad.reshape(-1)[at].item()


def test_gradient_of_a_gradient_is_refused(G):
    offsets, _ = offsets_of([2, 3])
    x, w = rand((5, 8), torch.bfloat16, 1).requires_grad_(), rand((2, 8, 8), torch.bfloat16, 2)
    with pytest.raises(RuntimeError, match="taken once"):
        torch.autograd.grad(G.product(x, w, offsets).sum(), x, create_graph=True)

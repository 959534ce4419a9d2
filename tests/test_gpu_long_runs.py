"""Sums over the longest runs and calls, of values of one sign that no type holds exactly, against fp64."""
import pytest
import torch

from tests.block_util import U32, half

pytestmark = pytest.mark.gpu
B, S = torch.bfloat16, torch.float32


def uniform(shape, dtype, seed):
    """Values of [1/2, 3/2)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for i in range(0, shape[0], 1 << 18):
        n = min(shape[0] - i, 1 << 18)
        out[i:i + n] = torch.rand((n, shape[1]), generator=g, device="cuda") + 0.5
    return out


def sums64(x, d):
    """(d^T x, sum of d) in fp64."""
    w = torch.zeros((d.shape[1], x.shape[1]), dtype=torch.float64, device="cuda")
    b = torch.zeros(d.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, x.shape[0], 1 << 17):
        x64, d64 = x[i:i + (1 << 17)].double(), d[i:i + (1 << 17)].double()
        w += d64.t().contiguous() @ x64
        b += d64.sum(0)
    return w, b


@pytest.mark.parametrize("P,N,K", [(1 << 23, 8, 8), (1 << 18, 4096, 4096)])      # 128 x 128 tiles; the persistent ones
@pytest.mark.parametrize("behind", [0, 3])
def test_gradients_of_one_long_run(P, N, K, behind):
    from bigrig_amd import grouped, lib
    lib.init(0)
    x, d = uniform((P, K), B, 1), uniform((P, N), B, 2)
    w, b = (torch.zeros(s, dtype=B, device="cuda", requires_grad=True) for s in ((2, N, K), (2, N)))
    offsets = torch.tensor([0, 0, P - behind], dtype=torch.int32, device="cuda")
    dw, db = torch.autograd.grad(grouped.product(x, w, offsets, b), (w, b), d)
    assert not dw[0].any() and not db[0].any()
    n, k = min(N, 48), min(K, 40)
    want_w, want_b = sums64(x[:P - behind, :k], d[:P - behind, :n])
    # The chains: 16 rows a matrix instruction, and a bias's every 64th row. Rounded to nearest, n steps of a growing sum are off
    # by 2^-24 sqrt(n) of it, eight times that taken; then the rounding to bf16. (Rounded toward zero, 2^19 steps would be off by
    # 2^-6, four bf16 roundings.)
    for got, want, steps in ((dw[1, :n, :k], want_w, P // 16), (db[1, :n], want_b, P // 64)):
        off = ((got.double() - want) / want).abs().max().item()
        assert off <= half(B) + 8 * U32 * steps ** 0.5, off


def test_column_sums_of_the_most_rows():
    from bigrig_amd import lib, norm
    lib.init(0)
    T, H = 1 << 23, 8
    y, r = (torch.full((T, H), v, dtype=B, device="cuda") for v in (1.5, 0.5))
    post, gate, nxt = (torch.full((H,), v, dtype=S, device="cuda", requires_grad=True) for v in (1.0, 0.75, 1.0))
    out = norm.leave(y, r, post, gate, 0.5, nxt)
    ones = torch.ones((T, H), dtype=B, device="cuda")
    got = torch.autograd.grad(out, (post, gate, nxt), (ones, ones))
    # Every row is one value, v = 1.5 or 0.875 (0.5 + 0.5 * 0.75 * 1): a norm of s = v / sqrt(v^2 + 1e-6), and the part of its
    # gradient that a row of equal gradients leaves, (1 - s^2) / sqrt(v^2 + 1e-6). A thread adds at most 2731 rows (four groups of
    # 768 blocks), then come 3, 48 and 15 sums; a row's value is off by 20 roundings.
    v = 0.875
    root = (v * v + 1e-6) ** 0.5
    D = 1.0 + (1.0 - (v / root) ** 2) / root
    u = 1.5 / (1.5 ** 2 + 1e-6) ** 0.5
    new = float(torch.tensor(0.5 + 0.375 * u).to(B))
    assert new == v
    for g, want in zip(got, (0.375 * D * u, 0.5 * u * D, v / root)):
        off = (g.double() / (T * want) - 1.0).abs().max().item()
        assert off <= (2731 + 3 + 48 + 15 + 20) * U32, off

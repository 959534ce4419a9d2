"""The persistent tiles of the grouped products where their last round is cut, and offsets that are out of order or range, on
the GPU."""
import ctypes as C

import pytest
import torch

from tests.block_util import rand
from tests.grouped_util import CUT, NARROW, WIDE
from tests.test_gpu_grouped import G, check  # noqa: F401

pytestmark = pytest.mark.gpu
B = torch.bfloat16


@pytest.mark.parametrize("dtype", [B, torch.float16])
@pytest.mark.parametrize("name", CUT)
@pytest.mark.parametrize("across", [False, True])
def test_a_cut_last_round(G, name, across, dtype):  # noqa: F811
    # (rounds and cuts of these calls: test_grouped_tiles.py)
    counts, behind, _, _ = CUT[name]
    N, K = (NARROW, WIDE) if across else (WIDE, NARROW)
    check(G, counts, N, K, dtype, bias=dtype == B, behind=behind, seed=len(counts))


GUARD = 1 << 16      # values on each side of an output


class Guarded:
    """An output inside a larger buffer whose other values are known."""

    def __init__(self, *shape):
        n = 1
        for s in shape:
            n *= s
        self.buf = torch.full((n + 2 * GUARD,), 7.0, dtype=B, device="cuda")
        self.out = self.buf[GUARD:GUARD + n].view(shape)

    def check(self, what):
        assert (self.buf[:GUARD] == 7).all() and (self.buf[GUARD + self.out.numel():] == 7).all(), what


def products(rows, weight, bias, dout, offsets):
    """The product and its gradients by the C-ABI, into guarded outputs."""
    from bigrig_amd import lib as L
    (P, K), (E, N, _) = rows.shape, weight.shape
    out, drows, dweight, dbias = Guarded(P, N), Guarded(P, K), Guarded(E, N, K), Guarded(E, N)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    lib = L.load()
    p = [t.data_ptr() for t in (rows, weight, bias, dout, off)]
    L.check(lib.brx_grouped_product(p[0], p[1], N * K, K, p[2], p[4], P, E, K, N, L.DT_BF16, out.out.data_ptr(), s))
    L.check(lib.brx_grouped_product_backward(p[3], p[0], p[1], N * K, K, p[4], P, E, K, N, L.DT_BF16, drows.out.data_ptr(),
                                             dweight.out.data_ptr(), dbias.out.data_ptr(), s))
    torch.cuda.synchronize()
    got = [out, drows, dweight, dbias]
    for g, what in zip(got, ("out", "drows", "dweight", "dbias")):
        g.check((what, offsets))
    return [g.out for g in got]


TOP, LOW = (1 << 31) - 1, -(1 << 31)
# of four experts; each form of the products: thin, 32, 64 and 128 rows a tile, persistent forward, backward and over the runs
SHAPES = [(8, 40, 72), (50, 40, 72), (150, 72, 136), (2000, 1032, 1096), (4500, 4104, 72), (4500, 72, 4104), (600, 2056, 2056)]


@pytest.mark.parametrize("P,N,K", SHAPES)
def test_offsets_of_any_kind_write_nothing_else(G, P, N, K):  # noqa: F811
    E = 4
    rows, weight, bias, dout = rand((P, K), B, 1), rand((E, N, K), B, 2), rand((E, N), B, 3), rand((P, N), B, 4)
    a, b, c = P // 5, P // 3, P // 2
    clean = products(rows, weight, bias, dout, [0, a, b, b, c])
    whole = products(rows, weight, bias, dout, [0, a, b, b, P])
    # the first offset is taken as 0, and one past the rows as their end
    for first in (5, a, TOP, LOW):
        assert all(torch.equal(x, y) for x, y in zip(products(rows, weight, bias, dout, [first, a, b, b, c]), clean)), first
    for last in (P + 1, 2 * P + 77, TOP):
        assert all(torch.equal(x, y) for x, y in zip(products(rows, weight, bias, dout, [0, a, b, b, last]), whole)), last
    # a negative one as 0, and a run that ends before it starts as empty
    less = products(rows, weight, bias, dout, [0, 0, b, b, c])
    assert all(torch.equal(x, y) for x, y in zip(products(rows, weight, bias, dout, [0, -9, b, b, c]), less))
    for x, y in zip(products(rows, weight, bias, dout, [0, c, b, b, c])[2:], clean[2:]):
        assert not x[1].any() and not x[2].any() and torch.equal(x[3], y[3])
    # overlapping runs: rows have one or another expert's value
    for o in ([0, P, 0, P, 0], [0, TOP, LOW, TOP, LOW], [TOP] * 5, [LOW] * 5, [0, P + 60, -5, P + 100, 1 << 30]):
        for t in products(rows, weight, bias, dout, o):
            assert torch.isfinite(t.float()).all(), o

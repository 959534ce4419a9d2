"""Sizes that the operators around a block's experts choose by themselves, without a GPU."""
import ctypes as C

import pytest

from bigrig_amd import lib as L


@pytest.mark.parametrize("T,H,blocks", [
    (1 << 20, 2048, 768), (1 << 20, 2049, 512), (1 << 20, 2880, 512), (1 << 20, 4096, 512), (1 << 20, 4097, 256), (1 << 20, 8192, 256),
    (300, 8192, 256), (200, 8192, 200), (600, 4096, 512), (400, 4096, 400), (700, 2048, 700), (3, 512, 1), (2000, 512, 500)])
def test_blocks_of_a_norm_gradient(T, H, blocks):
    # what its registers let run at once on 256 CUs: three blocks a CU, of wider rows two, one
    out = C.c_size_t()
    L.check(L.load().brx_norm_workspace_bytes(T, H, C.byref(out)))
    assert out.value == 3 * blocks * H * 4

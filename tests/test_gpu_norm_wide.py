"""Norm gradients of wide rows, several a block, against fp64."""
import pytest
import torch

from tests.test_gpu_norm import M, leave_case  # noqa: F401

pytestmark = pytest.mark.gpu
B, S = torch.bfloat16, torch.float32


@pytest.mark.parametrize("T,H,yd,rd", [(1100, 2056, B, S), (1030, 2880, B, B), (600, 4099, S, S), (520, 8192, B, B)])
def test_several_rows_a_block(M, T, H, yd, rd):  # noqa: F811
    leave_case(M, T, H, yd, rd, 1, "channel", 1, B)

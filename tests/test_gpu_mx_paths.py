"""The MXFP4 operators' kernels past the few-pair ones, and the limits of their calls, on the GPU."""
import ctypes as C

import pytest

from bigrig_amd import lib as L
from bigrig_amd.spec import GPT_OSS_120B
from tests.gpu_util import build_gpu_layer
from tests.helpers import make_layer, small

pytestmark = pytest.mark.gpu


def test_pairs_of_rows_past_32_bit_offsets_are_refused(gpu):
    """2^20 rows of 8192 values have 4 GB of codes: the pairs form refuses them as the product does, before it
    looks at the rows (the pointers are a small tensor's)."""
    import torch
    spec = small(GPT_OSS_120B, hidden=8192, inter=64, n_experts=2, top_k=1)
    _, _, pool, _ = build_gpu_layer(make_layer(spec, seed=5, expert_std=0.05), gpu)
    x = torch.zeros(1 << 16, dtype=torch.uint8, device=gpu)
    pair = torch.zeros(1, dtype=torch.int32, device=gpu)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    d, lib = spec.desc(), L.load()
    for T in (1 << 20, (1 << 31) - 1):
        rc = lib.brx_mx_moe_forward_pairs(C.byref(d), pool.device.handle, x.data_ptr(), T, pair.data_ptr(), pair.data_ptr(),
                                          None, 1, 1, None, x.data_ptr(), L.DT_BF16, 0, ws.data_ptr(), ws.numel(), None)
        assert rc == L.BRX_EINVAL and "2^32 - 256" in lib.brx_last_error().decode()
        rc = lib.brx_mx_expert_product(C.byref(d), pool.device.handle, x.data_ptr(), x.data_ptr(), T, pair.data_ptr(),
                                       pair.data_ptr(), None, 1, 1, 0, x.data_ptr(), ws.data_ptr(), ws.numel(), None)
        assert rc == L.BRX_EINVAL and "2^32 - 256" in lib.brx_last_error().decode()
    torch.cuda.synchronize()
    pool.close()

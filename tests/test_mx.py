"""MXFP4 rows and products without a GPU: what the calls refuse, the workspace arithmetic, and the 64-bit
restatement the GPU tests compare with against formats.quantize_mxfp4."""
import ctypes as C

import numpy as np
import pytest

from bigrig_amd import formats as F
from bigrig_amd import lib as L
from bigrig_amd import mx
from bigrig_amd.spec import E256_SHARED, GPT_OSS_120B, QWEN3_30B_A3B
from tests import mx_oracle as O
from tests.helpers import small

MX = F.QuantSpec(4, 32, "mxfp4")


def test_restatement_is_the_packers_quantizer():
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((40, 256)) * np.exp2(rng.integers(-20, 20, (40, 1)))).astype(np.float32)
    w[3, :32] = 0.0
    w[4, 32:64] = -0.0
    w = F.round_bf16(w)      # (bf16 values: the packer's fp32 log2 is exact enough on every one)
    wq, sc = F.quantize_mxfp4(w)
    codes, scales = O.quantize(w.astype(np.float64))
    assert np.array_equal(sc, scales)
    assert np.array_equal(wq.view(np.uint8).reshape(40, -1), O.pack(codes))


def test_ties_and_saturation():
    v = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -0.75, -5.0, -7.9])
    assert O.to_codes(v).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 0, 10, 14, 15]


def _err():
    return L.load().brx_last_error().decode()


@pytest.mark.parametrize("args, what", [
    ((0, 7, 1, 1, 32, 0, 32, 0, 0, 0, 0, None), "dtype"),
    ((0, L.DT_F32, 1, 1, 33, 0, 32, 0, 0, 0, 0, None), "multiple of 32"),
    ((0, L.DT_F32, -1, 1, 32, 0, 32, 0, 0, 0, 0, None), "negative"),
    ((0, L.DT_F32, 1, -5, 32, 0, 32, 0, 0, 0, 0, None), "negative"),
    ((0, L.DT_F32, 1 << 20, 1 << 20, 1 << 20, 0, 32, 0, 0, 0, 0, None), "2^40"),
])
def test_quantize_refuses(args, what):
    assert L.load().brx_mx_quantize(*args) == L.BRX_EINVAL
    assert what in _err()


def test_dequantize_refuses():
    lib = L.load()
    assert lib.brx_mx_dequantize(0, 0, 0, 0, 1, 1, 48, L.DT_F32, 0, None) == L.BRX_EINVAL
    assert "multiple of 32" in _err()
    assert lib.brx_mx_dequantize(0, 0, 0, 0, 1, 1, 64, 9, 0, None) == L.BRX_EINVAL


def _ws(spec, T, n, shared=0, product=0):
    out = C.c_size_t()
    d = spec.desc()
    rc = L.load().brx_mx_workspace_bytes(C.byref(d), T, n, shared, product, C.byref(out))
    return rc, out.value


def test_workspace_bytes():
    spec = small(E256_SHARED, quant=MX)
    rc, n = _ws(spec, 64, 512, 1)
    assert rc == 0
    # at least x and h rows and the down rows of every pair, routed and shared
    need = (64 * spec.hidden + 576 * spec.inter) * 17 // 32 + 576 * spec.hidden * 2
    assert need <= n < 2 * need
    assert _ws(spec, 64, 512)[1] < n
    assert _ws(spec, 64, 512, 0, 1)[1] < 64 * 1024
    assert _ws(spec, 0, 0)[0] == 0


def test_workspace_refusals():
    assert _ws(QWEN3_30B_A3B, 1, 8)[0] == L.BRX_EINVAL and "MXFP4 experts" in _err()
    assert _ws(GPT_OSS_120B, 1, 4, 1)[0] == L.BRX_EINVAL and "shared" in _err()
    assert _ws(GPT_OSS_120B, -1, 4)[0] == L.BRX_EINVAL and "negative" in _err()
    assert _ws(GPT_OSS_120B, 1, (1 << 21) + 1)[0] == L.BRX_EINVAL and "at most" in _err()
    d = GPT_OSS_120B.desc()
    assert L.load().brx_mx_workspace_bytes(C.byref(d), 1, 4, 0, 0, None) == L.BRX_EINVAL


def test_python_refusals_without_a_gpu():
    import torch
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="on the GPU"):
        mx.quantize(x)
    with pytest.raises(ValueError, match="on the GPU"):
        mx.dequantize(mx.MXRows(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)))
    with pytest.raises(ValueError, match="not mxfp4"):
        mx.pack_experts(QWEN3_30B_A3B, {})
    with pytest.raises(ValueError, match="projections"):
        mx.pack_experts(GPT_OSS_120B, {"fc1": x})
    spec = small(QWEN3_30B_A3B, quant=MX, hidden=64, inter=64, n_experts=4, top_k=2)
    w = {p: torch.zeros(4, 64, 64) for p in ("gate_proj", "up_proj", "down_proj")}
    with pytest.raises(ValueError, match="biases"):
        mx.pack_experts(spec, w, {"gate_proj": x})
    with pytest.raises(ValueError, match="up_proj"):
        mx.pack_experts(spec, dict(w, up_proj=torch.zeros(4, 64, 32)))
    with pytest.raises(ValueError, match="bfloat16"):
        mx.moe_forward(spec, None, torch.zeros(1, 64), None)
    with pytest.raises(ValueError, match="MXFP4 experts"):
        mx.moe_forward(QWEN3_30B_A3B, None, x, None)
    with pytest.raises(ValueError, match="projection"):
        mx.expert_product(spec, None, None, None, None, "fc1")


def test_matrices_of_strided_tensors():
    import torch
    t = torch.zeros(4, 6, 64)
    assert mx._matrices(t, "t") == (1, 24, 0, 64)
    assert mx._matrices(t[:, ::2], "t") == (4, 3, 384, 128)
    assert mx._matrices(t[:, :, :32], "t") == (4, 6, 384, 64)
    assert mx._matrices(t[0, 0], "t") == (1, 1, 0, 0)
    assert mx._matrices(t[:0], "t") == (0, 0, 0, 0)
    assert mx._matrices(torch.zeros(2, 4, 6, 64)[:, :, ::2], "t") == (8, 3, 384, 128)
    with pytest.raises(ValueError, match="innermost"):
        mx._matrices(t.transpose(1, 2), "t")
    with pytest.raises(ValueError, match="collapse"):
        mx._matrices(torch.zeros(4, 4, 6, 64)[:, ::3, ::2], "t")
    with pytest.raises(ValueError, match="dimensions"):
        mx._matrices(torch.zeros(()), "t")


def test_switch_refuses_activations():
    from bigrig_amd.layer import StreamingSwitchGLU

    class Pool:
        spec = QWEN3_30B_A3B
    with pytest.raises(ValueError, match="activations"):
        StreamingSwitchGLU(Pool(), None, activations="fp8")
    with pytest.raises(ValueError, match="MXFP4 experts"):
        StreamingSwitchGLU(Pool(), None, activations="mxfp4")
    Pool.spec = GPT_OSS_120B
    assert StreamingSwitchGLU(Pool(), None, activations="mxfp4").activations == "mxfp4"


def test_rows_past_32_bit_offsets_are_refused():
    """Activations whose codes pass 4 GB, which the kernels' offsets do not reach: refused by size, whatever the
    form of the call, and the widest that fit are not."""
    import torch
    spec = small(GPT_OSS_120B, hidden=8192, inter=64, n_experts=4, top_k=2)
    most = mx.MAX_CODES // 4096
    assert most == (1 << 20) - 1
    assert _ws(spec, most, 8)[0] == 0
    assert _ws(spec, most + 1, 8)[0] == L.BRX_EINVAL and "2^32 - 256" in _err()
    assert _ws(spec, most + 1, 0)[0] == 0            # (no pairs: nothing is addressed)
    i32 = torch.empty(8, dtype=torch.int32, device="meta")
    for T in (most + 1, 1 << 31, (1 << 32) + 5):     # (the last two have other values in 32 bits)
        rows = mx.MXRows(torch.empty(T, 4096, dtype=torch.uint8, device="meta"),
                         torch.empty(T, 256, dtype=torch.uint8, device="meta"))
        with pytest.raises(ValueError, match="rows of 8192 values"):
            mx.expert_product(spec, None, rows, i32, i32, "gate_proj")
        with pytest.raises(ValueError, match="rows of 8192 values"):
            mx.forward_pairs(spec, None, torch.empty(T, 8192, dtype=torch.bfloat16, device="meta"), i32, i32, None,
                             None, 0)
    with pytest.raises(ValueError, match="tokens"):
        mx.moe_forward(spec, None, torch.empty(mx.MAX_TOKENS + 1, 8192, dtype=torch.bfloat16, device="meta"), None)
    many = torch.empty(mx.MAX_PAIRS + 1, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="pairs in one call"):
        mx.forward_pairs(spec, None, torch.empty(4, 8192, dtype=torch.bfloat16, device="meta"), many, many, None, None, 0)


def test_workspace_of_rows_has_no_rows_to_sum():
    """Unreduced rows and the pairs form write where the caller says: no fp32 row a pair in their scratch."""
    spec = small(E256_SHARED, quant=MX)
    for T, shared in ((64, 0), (2048, 0), (2048, 1)):
        pairs = T * spec.top_k
        sums, rows = _ws(spec, T, pairs, shared, L.MX_LAYER)[1], _ws(spec, T, pairs, shared, L.MX_ROWS)[1]
        assert sums - rows == (pairs + shared * T) * spec.hidden * 4
        # x and h rows, four bytes a pair and the tile list
        assert rows < (T * spec.hidden + (pairs + T) * spec.inter) * 17 // 32 + 64 * (pairs + T) + 64 * 1024
    assert _ws(spec, 64, 512, 0, 3)[0] == L.BRX_EINVAL and "call 3" in _err()
    assert _ws(spec, 64, 512, 0, -1)[0] == L.BRX_EINVAL

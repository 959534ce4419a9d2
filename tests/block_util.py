"""Shared by the tests of the operators around a block's experts: inputs and error bounds.

A bound counts roundings: `half(t)` is half a step of type t relative to a value, U32 that of fp32; a sum of n
terms in fp32, in any order, is off by at most n U32 times the sum of the terms' magnitudes (to first order;
SUM_U is twice that, which also covers a matrix instruction that rounds its partial sums toward zero)."""
import torch

U32 = 2.0 ** -24
SUM_U = 2.0 ** -23
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    """Half the least step of a type: what a rounding may be off by at values below its normal range."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, want, slack, what=""):
    """got (of its type) is want (fp64) up to `slack` (fp64, absolute, what the fp32 steps may be off by) and one rounding."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    g = got.detach().double().cpu()
    want, slack = want.double().cpu(), torch.as_tensor(slack, dtype=torch.float64).cpu()
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(g), bad), f"{what}: NaN in other places"
    lim = slack + half(got.dtype) * (want.abs() + slack) + tiny(got.dtype)
    off = torch.where(bad, torch.zeros_like(g), (g - want).abs())
    worst = (off - lim).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: off by {worst:.3e} more than its bound (largest error {off.max().item():.3e})"


def rand(shape, dtype, seed, dev="cuda", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(dev)


def routing(T, k, E, seed, drop=0.0, dev="cuda"):
    """int32 [T, k]: distinct experts a token where E allows it, some pairs dropped."""
    g = torch.Generator().manual_seed(seed)
    if k <= E:
        idx = torch.rand((T, E), generator=g).argsort(-1)[:, :k].int() if T else torch.zeros((0, k), dtype=torch.int32)
    else:
        idx = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    if drop:
        idx = torch.where(torch.rand((T, k), generator=g) < drop, -1, idx)
    return idx.contiguous().to(dev)

"""Inputs and 64-bit references for the tests of the linear layers with an epilogue and of the layers of experts.

Where a test wants equality it takes numbers whose sums are exact in fp32 whatever their order: whole activations up to 4,
scales of 1/64, 1/128 and 1/256. A product is then a whole multiple of 2^-8 of at most 60 / 64, so that sums over up to 17408
columns stay below 2^22 multiples, bias and residual (whole, up to 64: 2^14 multiples) included: below 2^24, no sum rounds.
"""
import numpy as np
import torch

GROUP = 128


def disk(rows, cols, seed, exact=True):
    """Checkpoint tensors of a layer on the GPU: packed codes, scales, zero points."""
    gen = torch.Generator().manual_seed(seed)
    packed = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, cols // 8), dtype=torch.int32, generator=gen)
    zp = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows // 8, cols // GROUP), dtype=torch.int32, generator=gen)
    if exact:
        scale = 2.0 ** -torch.randint(6, 9, (rows, cols // GROUP), generator=gen).float()
    else:
        scale = torch.randn((rows, cols // GROUP), generator=gen).abs() * 0.02 + 1e-4
    return packed.cuda(), scale.to(torch.bfloat16).cuda(), zp.cuda()


def weights64(packed, scale, zp):
    """bf16((q - zp) * scale) of every element, in fp64."""
    at = torch.arange(0, 32, 4, device=packed.device)
    q = (packed.long().unsqueeze(-1) >> at & 15).flatten(1)
    z = (zp.long().unsqueeze(1) >> at[:, None] & 15).flatten(0, 1)
    w = (q - z.repeat_interleave(GROUP, 1)).double() * scale.double().repeat_interleave(GROUP, 1)
    return w.to(torch.bfloat16).double()


def whole(shape, limit, seed):
    """Whole numbers up to `limit` in bf16."""
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-limit, limit + 1, shape, generator=gen).to(torch.bfloat16).cuda()


def activate64(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(-v / 2 ** 0.5)
    if act == "gelu_tanh":
        # 0.5 (1 + tanh u) = sigmoid(2 u); as written it would cancel for negative u, in 64 bits too (u = -20: 4e-18 beside 1)
        return v * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    if act == "swiglu":
        g, u = v.chunk(2, dim=-1)
        return g * torch.sigmoid(g) * u
    return v


def code(pkg, act):
    return {"none": pkg.ACT_NONE, "silu": pkg.ACT_SILU, "gelu": pkg.ACT_GELU, "gelu_tanh": pkg.ACT_GELU_TANH,
            "swiglu": pkg.ACT_SWIGLU}[act]


def assert_close_to_rounding(got, ref64, act):
    """`got` (bf16) against exact sums in 64 bits. Without an activation it is the correctly rounded value. With one, what is rounded
    differs from the exact value by the device's exp (2 units in 2^-24 and 2^-24 |v| for the scaled argument, |v| < 128: 2^-16), the
    division and the products (a few 2^-24 each) or erfc (under 2^-20): 2^-15 relative in all. Rounding to bf16 adds at most 2^-8."""
    if act == "none":
        assert torch.equal(got, ref64.to(torch.bfloat16))
        return
    err = (got.double() - ref64).abs()
    # (values under 2^-100 are zero for this purpose: a gate of -80 and below)
    bad = err > ref64.abs() * (2.0 ** -8 + 2.0 ** -15) + 2.0 ** -100
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, worst {float((err / (ref64.abs() + 1e-30))[bad].max()):.3g}"

"""Hidden values of the mixture-of-experts layer, one at a time: how many bits of them the down product sees."""
import math

import pytest
import torch

import h100_gemm_b200 as g

BF16, FP16 = torch.bfloat16, torch.float16
KINDS = ["bf16", "fp16", "mxfp4", "nvfp4"]


def matrix(values, kind):
    """A [rows, cols] matrix of -1, 0 and 1 as the layer takes it."""
    if kind in ("bf16", "fp16"):
        return values.to(BF16 if kind == "bf16" else FP16).cuda()
    code = torch.where(values == 0, 0, torch.where(values > 0, 2, 10)).to(torch.uint8)
    blocks = -(-values.shape[1] // (32 if kind == "mxfp4" else 16))
    scale = torch.full((values.shape[0], blocks), 127 if kind == "mxfp4" else 0x38, dtype=torch.uint8)  # 1
    return g.MxTensor.from_parts((code[:, 0::2] | code[:, 1::2] << 4).cuda(), scale.cuda(), values.shape[1], kind)


def layer(x, down, kind):
    """The layer whose hidden value i is silu(x[i]) * x[I + i]: one expert beside a masked one, so its weight is 1."""
    I = down.shape[1]
    H = 2 * I
    up = torch.zeros(2, 2 * I, H)
    up[1] = torch.eye(H)
    rows = torch.zeros(2, H, I)
    rows[1, :down.shape[0]] = down
    w1, w2 = matrix(up.view(-1, H), kind), matrix(rows.view(-1, I), kind)
    if kind in ("bf16", "fp16"):
        w1, w2 = w1.view(2, H, H), w2.view(2, H, I)
    bias = torch.tensor([-math.inf, 0.0]).cuda()
    out, ids, weights = g.moe_layer(x, torch.zeros(2, H, dtype=x.dtype).cuda(), w1, w2, 1, bias=bias, return_routing=True)
    assert (ids == 1).all() and (weights[x.isfinite().all(1)] == 1).all()  # (a NaN logit's weight is exp(NaN) / exp(NaN))
    return out[:, :down.shape[0]]


def silu(v):
    return v * torch.sigmoid(v)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 13])
@pytest.mark.parametrize("kind", KINDS)
def test_down_product_sees_the_bits_of_fp32(kind, T):
    """Rows of the down product take two 16-bit numbers off a hidden value, its nearest one and the nearest one of
    the rest: what is left shows the bits behind those 16 (bf16) or 22 (fp16).

    Off by, relative to the hidden value: the exponential 2^-23, sum, division and product 3 x 2^-24, 22 bits kept 2^-22, the
    sums of three terms 6 x 2^-24: 15 x 2^-24, below 2^-20; and half a step of the output."""
    dtype = FP16 if kind == "fp16" else BF16
    n = 88
    gen = torch.Generator().manual_seed(T)
    gate = (torch.rand(T, n, generator=gen) * 9 - 3).to(dtype)
    up = (torch.rand(T, n, generator=gen) * 1.5 + 0.5).to(dtype)
    h = silu(gate.double()) * up.double()
    one = h.to(dtype)
    two = (h - one.double()).to(dtype)
    # silu(32) is 32 to 2^-45
    gates = torch.stack([gate, torch.full_like(gate, 32.0), torch.full_like(gate, 32.0)], 2)
    ups = torch.stack([up, (one.float() / 32).to(dtype), (two.float() / 32).to(dtype)], 2)
    down = torch.zeros(n, 3 * n)
    for r in range(n):
        down[r, 3 * r], down[r, 3 * r + 1], down[r, 3 * r + 2] = 1, -1, -1
    out = layer(torch.cat([gates.view(T, -1), ups.view(T, -1)], 1).cuda(), down, kind).double().cpu()
    want = h - 32 * ups[:, :, 1].double() - 32 * ups[:, :, 2].double()
    bound = 2.0 ** -20 * h.abs() + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = (out - want).abs()
    assert (off <= bound).all(), f"{(off > bound).sum()} of {off.numel()} outside, up to {(off / h.abs()).max():.2g} of the value"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "mxfp4", "nvfp4"])
def test_infinite_and_nan_hidden_values(kind):
    """A hidden value beyond fp32 is infinite, and so is a sum of those; a NaN stays one, in its token alone."""
    x = torch.full((3, 48), 2.0 ** 100, dtype=BF16)
    x[1, 24:] = -2.0 ** 100
    x[2] = 1.0
    x[2, 3] = math.nan
    out = layer(x.cuda(), torch.ones(8, 24), kind)
    assert (out[0] == math.inf).all() and (out[1] == -math.inf).all() and out[2].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 7])
@pytest.mark.parametrize("size", [2.0 ** -8, 2.0 ** -12, 2.0 ** -15])
def test_small_fp16_hidden_values(size, T):
    """Small hidden values (a routing weight of a hundredth is enough) under large down weights: the rest behind the
    nearest fp16 number is far below fp16's smallest one.

    Off by: 2^-20 as above, and 2^-36 where that rest is subnormal; 1024 times that, and half a step of the output."""
    n = 64
    gen = torch.Generator().manual_seed(T)
    gate = (torch.rand(T, n, generator=gen) * 4 + 1).to(FP16)
    up = ((torch.rand(T, n, generator=gen) + 0.5) * size).to(FP16)
    h = silu(gate.double()) * up.double()
    near = (h / 32).to(FP16)                                   # 32 times it is taken off, so that the rest shows
    gates = torch.stack([gate, torch.full_like(gate, 32.0)], 2)
    ups = torch.stack([up, near], 2)
    down = torch.zeros(n, 2 * n)
    for r in range(n):
        down[r, 2 * r], down[r, 2 * r + 1] = 1024, -1024
    out = layer(torch.cat([gates.view(T, -1), ups.view(T, -1)], 1).cuda(), down, "fp16").double().cpu()
    want = 1024 * (h - 32 * near.double())
    bound = 1024 * (2.0 ** -20 * h + 2.0 ** -36) + 2.0 ** -11 * want.abs() + 2.0 ** -25
    off = (out - want).abs()
    assert (off <= bound).all(), f"{(off > bound).sum()} of {off.numel()} outside, up to {(off / bound).max():.2g} times the bound"

"""The expert layer on the ways through its kernels that ordinary small sizes miss."""
import pytest
import torch

from test_moe import BF16, FP16, check, make
from test_mx import E4M3, random_mx

# hidden sizes beyond one step of eight warps (2048), with one and more MMA tiles of tokens per expert, and steps that the end of the rows
# cuts short after a whole one
LONG = [(1, 4, 2, 4096, 64), (3, 4, 2, 4096, 72), (9, 2, 2, 2056, 24), (20, 3, 2, 2312, 520), (41, 6, 3, 4104, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, FP16, "mxfp4", "nvfp4"])
@pytest.mark.parametrize("T,E,k,H,I", LONG)
def test_hidden_sizes_of_several_steps(T, E, k, H, I, kind):
    fmt = kind if isinstance(kind, str) else None
    check(*make(T, E, H, I, BF16 if fmt else kind, T + H, fmt), k)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("T", [32, 33, 40, 41])
def test_sums_of_one_and_of_two_units(T, fmt):
    """Up to 40 tokens 4-bit experts have room for the sums of two units; several units per CTA use them in turn."""
    check(*make(T, 64, 128, 264, BF16, T, fmt), 8)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 11])
@pytest.mark.parametrize("low,high", [(0, 0), (1, 1), (1, 7), (8, 15), (0x77, 0x7E), (0x7E, 0x7E), (0, 126)])
def test_nvfp4_experts_with_scales_of_any_size(low, high, T):
    """Block scales from the smallest subnormal, 2^-9, to 448; the tensor scale keeps sums of ordinary size."""
    E, k, H, I = 3, 2, 328, 72
    top = max(float(E4M3[high]), 2.0 ** -9)
    ts = 2.0 ** -round(torch.tensor(top).log2().item() + 4)
    x, router, *_ = make(T, E, H, I, BF16, 5)
    w1, v1 = random_mx(E * 2 * I, H, "nvfp4", 1, low, high, ts)
    w2, v2 = random_mx(E * H, I, "nvfp4", 2, low, high, ts)
    check(x, router, w1, w2, torch.from_numpy(v1).view(E, 2 * I, H), torch.from_numpy(v2).view(E, H, I), k)

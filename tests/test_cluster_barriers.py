"""Cluster barriers behind loops whose trip counts differ between the lanes of a warp."""
import re
from pathlib import Path

import pytest
import torch

import h100_gemm_b200 as g

SM100 = Path(g.__file__).resolve().parent / "csrc" / "sm100"


def test_lanes_meet_before_every_aligned_cluster_barrier():
    """The aligned barrier is undefined for a warp that arrives in parts; only the two wrappers issue it."""
    issued = 0
    for path in sorted(SM100.glob("*.cuh")):
        text = path.read_text()
        for m in re.finditer(r'asm volatile\("barrier\.cluster\.\w+\.\w+\.aligned', text):
            issued += 1
            assert path.name == "ptx.cuh", f"{path.name} issues a cluster barrier by itself"
            assert text[:m.start()].rstrip().endswith("__syncwarp();"), m.group(0)
    assert issued == 2


def test_lanes_meet_before_the_expert_layers_mmas():
    """mma.sync.aligned is undefined for a warp in parts, and sums are written lane by lane under conditions before it."""
    text = (SM100 / "moe.cuh").read_text()
    calls = list(re.finditer(r"\n    w\.mma_(tokens|hidden)\(", text))
    assert len(calls) == 2
    for m in calls:
        assert "__syncwarp();" in text[:m.start()].rsplit("\n", 1)[1], m.group(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 2, 3, 5, 7])
def test_experts_whose_sums_leave_warps_part_filled(T, dtype):
    """T * 17 sums to join and T * 16 outputs over clusters of up to eight CTAs: no multiple of 32."""
    E, k, H, I = 16, 4, 72, 1032
    gen = torch.Generator().manual_seed(T)
    draw = lambda *s: (torch.randint(-1, 2, s, generator=gen)).to(dtype).cuda()  # noqa: E731
    x, w1, w2 = draw(T, H), draw(E, 2 * I, H), draw(E, H, I)
    w1[:, :I] = 0
    w1[:, :I, 0] = 1
    x[:, 0] = 32            # every gate is 32, so silu is 32 to the last bit of fp32
    w1[:, I:, 0] = 0
    bias = torch.full((E,), -float("inf"))
    bias[3] = 0.0           # one expert: its weight is 1
    out = g.moe_layer(x, torch.zeros(E, H, dtype=dtype, device="cuda"), w1, w2, k, bias=bias.cuda())
    hidden = 32 * (x.double() @ w1[3, I:].double().T)      # whole multiples of 32, at most 32 * 71: exact in either type's parts
    want = (hidden @ w2[3].double().T).to(dtype)           # sums below 2^24
    assert torch.equal(out, want)

"""Experts that a bias of -inf takes out, beside infinities and NaN."""
import math

import pytest
import torch

import h100_gemm_b200 as g

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_experts_stay_out_whatever_they_hold(bad, dtype, renormalize):
    """Slots that hold no expert yet: router rows and weights full of rubbish, taken out by the bias."""
    T, E, k, H, I = 6, 12, 3, 136, 40
    gen = torch.Generator().manual_seed(7)
    draw = lambda *s: (torch.randn(*s, generator=gen) * s[-1] ** -0.5).to(dtype).cuda()  # noqa: E731
    x, router, w1, w2 = draw(T, H), draw(E, H), draw(E, 2 * I, H), draw(E, H, I)
    bias = torch.randn(E, generator=gen).cuda()
    bias[[0, 5, 11]] = -math.inf
    want = g.moe_layer(x, router, w1, w2, k, bias=bias, renormalize=renormalize, return_routing=True)
    for t in (router, w1, w2):
        t[[0, 5, 11]] = bad
    got = g.moe_layer(x, router, w1, w2, k, bias=bias, renormalize=renormalize, return_routing=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # nobody left: no expert, zeros
    out, ids, weights = g.moe_layer(x, router, w1, w2, k, bias=torch.full_like(bias, -math.inf), renormalize=renormalize,
                                    return_routing=True)
    assert not out.any() and (ids == -1).all() and not weights.any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_token_that_is_not_finite_does_not_reach_a_masked_expert(bad):
    T, E, k, H, I = 3, 9, 4, 64, 24
    gen = torch.Generator().manual_seed(8)
    draw = lambda *s: (torch.randn(*s, generator=gen) * s[-1] ** -0.5).to(BF16).cuda()  # noqa: E731
    x, router, w1, w2 = draw(T, H), draw(E, H), draw(E, 2 * I, H), draw(E, H, I)
    bias = torch.zeros(E, device="cuda")
    bias[:4] = -math.inf
    x[1, 2] = bad
    _, ids, _ = g.moe_layer(x, router, w1, w2, k, bias=bias, return_routing=True)
    assert (ids[[0, 2]] >= 4).all()
    assert ((ids[1] >= 4) | (ids[1] == -1)).all()      # (a product of -inf takes its expert out as well)
    assert len(set(ids[1][ids[1] >= 0].tolist())) == (ids[1] >= 0).sum()

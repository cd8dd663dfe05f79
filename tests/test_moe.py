"""The mixture-of-experts layer against its formula in 64 bits, expert by expert and token by token."""
import math

import pytest
import torch

import h100_gemm_b200 as g
from h100_gemm_b200 import api, moe
from test_mx import random_mx

BF16, FP16 = torch.bfloat16, torch.float16


def route_ref(logits, k, renormalize):
    """ids and weights from [T, E] float64 logits: stable order, NaN first, -inf never."""
    T, E = logits.shape
    ids = torch.full((T, k), -1, dtype=torch.int32)
    weights = torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        row = logits[t].tolist()
        order = sorted((e for e in range(E) if row[e] != -math.inf),
                       key=lambda e: (0, 0.0, e) if math.isnan(row[e]) else (1, -row[e], e))[:k]
        over = order if renormalize else [e for e in range(E) if row[e] != -math.inf]
        p = torch.softmax(torch.tensor([row[e] for e in over], dtype=torch.float64), 0) if over else None
        for j, e in enumerate(order):
            ids[t, j] = e
            weights[t, j] = p[over.index(e)]
    return ids, weights


def layer_ref(x, ids, weights, w1, w2):
    """out and the sums of magnitudes its rounding errors are measured by, in 64 bits. h's magnitudes: what each
    hidden value may be off by is bounded through |d silu| <= 1.1, |silu(a)| <= |a|."""
    T, H = x.shape
    E, I = w1.shape[0], w2.shape[2]
    out, size, up_err = (torch.zeros(T, H, dtype=torch.float64) for _ in range(3))
    x = x.double().cpu()
    for e in range(E):
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        if not len(t):
            continue
        a, b, d = w1[e, :I].double().cpu(), w1[e, I:].double().cpu(), w2[e].double().cpu()
        gate, up = x[t] @ a.T, x[t] @ b.T
        p = weights[t, slot][:, None].double()
        h = p * gate * torch.sigmoid(gate) * up
        out[t] += h @ d.T
        size[t] += h.abs() @ d.abs().T
        # fp32 sums of H products: an error of 2^-22 of the magnitudes for each of H / 16 MMAs and 16 joins
        tol = (H / 16 + 16) * 2.0 ** -22
        gate_off, up_off = tol * (x[t].abs() @ a.abs().T), tol * (x[t].abs() @ b.abs().T)
        silu = (gate * torch.sigmoid(gate)).abs()
        up_err[t] += (p * (1.1 * gate_off * up.abs() + silu * up_off + 1.1 * gate_off * up_off)) @ d.abs().T
    return out, size, up_err


def allowed(dtype, out, size, up_err, I, top_k):
    """|kernel - formula|: the output's rounding, h's rounding to two 16-bit parts (the square of one's), 2^-20 for its fp32
    factors (weight, sigmoid, products), fp32 sums of the down product, and what gate and up bring along. fp16's
    parts may be subnormal: 2^-25 each."""
    eps = torch.finfo(dtype).eps / 2
    return eps * out.abs() + (eps ** 2 + 2.0 ** -20 + (2 * top_k * I / 16 + 80) * 2.0 ** -22) * size + up_err + 1e-6 * (dtype == FP16) + 1e-30


def make(T, E, H, I, dtype, seed, fmt=None):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=gen).to(dtype).cuda()
    router = (torch.randn(E, H, generator=gen) * H ** -0.5).to(dtype).cuda()
    if fmt:
        low, high, ts = (120, 123, 1.0) if fmt == "mxfp4" else (0x18, 0x48, 2.0 ** -5)
        w1, v1 = random_mx(E * 2 * I, H, fmt, seed + 1, low, high, ts)
        w2, v2 = random_mx(E * H, I, fmt, seed + 2, low, high, ts)
        return x, router, w1, w2, torch.from_numpy(v1).view(E, 2 * I, H), torch.from_numpy(v2).view(E, H, I)
    w1 = (torch.randn(E, 2 * I, H, generator=gen) * H ** -0.5).to(dtype).cuda()
    w2 = (torch.randn(E, H, I, generator=gen) * I ** -0.5).to(dtype).cuda()
    return x, router, w1, w2, w1, w2


def check(x, router, w1, w2, v1, v2, k, bias=None, renormalize=True, ids_known=True):
    out, ids, weights = g.moe_layer(x, router, w1, w2, k, bias=bias, renormalize=renormalize, return_routing=True)
    logits = x.double().cpu() @ router.double().cpu().T
    if bias is not None:
        logits = logits + bias.double().cpu()
    want_ids, want_w = route_ref(logits, k, renormalize)
    if ids_known:
        assert torch.equal(ids.cpu(), want_ids)
        # logits off by (H / 64 + 8) 2^-24 of their magnitudes, the exponential, sum and division by a few units
        mag = (x.double().cpu().abs() @ router.double().cpu().abs().T).max().item()
        rel = 4 * (x.shape[1] / 64 + 8) * 2.0 ** -24 * mag + 64 * 2.0 ** -24
        assert ((weights.double().cpu() - want_w).abs() <= rel * want_w).all()
    ref, size, up_err = layer_ref(x, ids.cpu(), weights.cpu(), v1, v2)
    bound = allowed(x.dtype, ref, size, up_err, w2.cols if isinstance(w2, g.MxTensor) else w2.shape[2], k)
    bad = ~((out.double().cpu() - ref).abs() <= bound)
    assert not bad.any(), f"{bad.sum()} of {bad.numel()} outside, first {bad.nonzero()[:4].tolist()}"
    assert torch.equal(out, g.moe_layer(x, router, w1, w2, k, bias=bias, renormalize=renormalize))  # bit for bit again
    return out, ids, weights


# --------------------------------------------------------------------------------------- no GPU
def test_workspace_and_refusals_without_a_device():
    lib = api.library()
    assert g.moe_workspace_bytes(1, 8, 2, 64, 64) == 512 + 2 * 256
    assert g.moe_workspace_bytes(64, 128, 8, 2048, 768) == 64 * 8 * 768 * 4 + 2 * 64 * 8 * 4
    for bad in ((0, 8, 2, 64, 64), (65, 8, 2, 64, 64), (1, 513, 2, 64, 64), (1, 8, 9, 64, 64), (1, 64, 33, 64, 64),
                (1, 8, 0, 64, 64), (1, 8, 2, 60, 64), (1, 8, 2, 64, 0)):
        assert g.moe_workspace_bytes(*bad) == 0
    for T, k, I in ((1, 1, 8), (3, 5, 40), (64, 32, 1000), (17, 3, 768), (8, 8, 64)):
        assert moe._workspace_bytes(T, k, I) == g.moe_workspace_bytes(T, 40, k, 64, I)
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    good = dict(x=z(2, 64), router=z(8, 64), w_gate_up=z(8, 64, 64), w_down=z(8, 64, 32), top_k=2)
    for change, text in ((dict(), "CUDA tensor"), (dict(x=z(2, 64, dtype=torch.float32)), "bfloat16 or float16"),
                         (dict(x=z(0, 64)), "tokens"), (dict(x=z(65, 64)), "tokens"), (dict(router=z(8, 32)), "router"),
                         (dict(top_k=9), "top_k"), (dict(top_k=0), "top_k"), (dict(w_gate_up=z(8, 62, 64)), "w_gate_up"),
                         (dict(w_down=z(8, 64, 31), w_gate_up=z(8, 62, 64)), "multiples of 8"),
                         (dict(w_down=z(8 * 64, 32)), "experts"), (dict(router=z(513, 64)), "experts")):
        with pytest.raises(g.GemmError, match=text):
            g.moe_layer(**{**good, **change})


def test_refusals_of_the_c_abi():
    lib = api.library()
    p = 4096

    def call(**kw):
        a = {**dict(f16=0, T=2, E=8, k=2, H=64, I=32, x=p, r=p, b=None, fmt=-1, w1=p, s1=None, w2=p, s2=None, out=p, ids=None,
                    wts=None, ws=p, n=1 << 20), **kw}
        return lib.b200_moe_layer(a["f16"], a["T"], a["E"], a["k"], a["H"], a["I"], a["x"], a["r"], a["b"], a["fmt"], a["w1"],
                                  a["s1"], 1.0, a["w2"], a["s2"], 1.0, 1, a["out"], a["ids"], a["wts"], a["ws"], a["n"], None)

    for kw in (dict(T=0), dict(T=65), dict(E=513), dict(k=9), dict(H=60), dict(I=0), dict(x=None), dict(r=None), dict(w1=None),
               dict(w2=None), dict(out=None), dict(x=p + 8), dict(w1=p + 2), dict(out=p + 1), dict(b=p + 2), dict(ids=p + 1),
               dict(fmt=2), dict(fmt=0), dict(fmt=0, s1=p, s2=p, f16=1), dict(ws=p + 16)):
        assert call(**kw) == api.STATUS_INVALID_ARG, kw
    for kw in (dict(ws=None), dict(n=10)):
        assert call(**kw) == api.STATUS_WORKSPACE, kw


# --------------------------------------------------------------------------------------- on the GPU
SIZES = [(1, 8, 2, 64, 32), (1, 64, 6, 512, 256), (2, 3, 3, 8, 8), (3, 16, 4, 264, 136), (7, 31, 5, 1000, 88), (8, 128, 8, 256, 64),
         (9, 8, 1, 2048, 40), (16, 2, 2, 128, 520), (17, 40, 8, 328, 64), (33, 12, 3, 136, 264), (64, 16, 4, 512, 128),
         (64, 1, 1, 72, 80), (64, 512, 32, 64, 8), (5, 500, 17, 104, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,E,k,H,I", SIZES)
def test_layer(T, E, k, H, I, dtype):
    check(*make(T, E, H, I, dtype, T + E + H), k)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("T,E,k,H,I", SIZES)
def test_layer_with_4_bit_experts(T, E, k, H, I, fmt):
    check(*make(T, E, H, I, BF16, T + E + H, fmt), k)


@pytest.mark.gpu
@pytest.mark.parametrize("byte", [0, 1, 59, 127, 128, 129, 200, 240])
def test_layer_4_bit_scales_of_any_size(byte):
    """Block scales from 2^-127 to 2^113, undone by the other matrix or the tokens, so that sums stay in range."""
    T, E, k, H, I = 3, 2, 2, 64, 32
    x, router, *_ = make(T, E, H, I, BF16, 3)
    other = min(254, max(0, 254 - byte)) if byte in (127, 128, 129) else 127
    x = (x * 2.0 ** min(100, max(-100, 127 - byte))).to(BF16)  # gate and up of ordinary size
    w1, v1 = random_mx(E * 2 * I, H, "mxfp4", 1, byte, byte)
    w2, v2 = random_mx(E * H, I, "mxfp4", 2, other, other)
    check(x, torch.zeros_like(router), w1, w2, torch.from_numpy(v1).view(E, 2 * I, H), torch.from_numpy(v2).view(E, H, I), k)


@pytest.mark.gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T", [1, 13])
def test_masked_experts_and_ties(T, renormalize):
    x, router, w1, w2, v1, v2 = make(T, 24, 128, 64, BF16, 11)
    bias = torch.randn(24, generator=torch.Generator().manual_seed(1)).cuda()
    bias[::2] = -math.inf
    check(x, router, w1, w2, v1, v2, 5, bias, renormalize)
    check(x, router, w1, w2, v1, v2, 16, bias, renormalize)          # more choices than experts that are left
    out, ids, weights = check(x, router, w1, w2, v1, v2, 4, torch.full((24,), -math.inf).cuda(), renormalize)
    assert not out.any() and (ids == -1).all() and not weights.any()  # nobody left: zeros
    _, ids, weights = check(x, torch.zeros_like(router), w1, w2, v1, v2, 6, None, renormalize)
    assert (ids.cpu() == torch.arange(6)).all()                       # ties: the lower index
    assert torch.allclose(weights, torch.full_like(weights, 1 / 6 if renormalize else 1 / 24), rtol=1e-6)
    lowest = torch.full((24,), torch.finfo(torch.float32).min).cuda()  # a mask of the type's lowest value is still a number
    _, ids, _ = check(x, router, w1, w2, v1, v2, 3, lowest, renormalize, ids_known=False)
    assert (ids >= 0).all()


@pytest.mark.gpu
def test_nan_token_stays_alone():
    x, router, w1, w2, v1, v2 = make(12, 16, 256, 64, BF16, 21)
    _, ids, weights = g.moe_layer(x, router, w1, w2, 3, return_routing=True)
    keep = torch.arange(12) != 5
    ref, size, up_err = layer_ref(x[keep], ids.cpu()[keep], weights.cpu()[keep], v1, v2)
    bound = allowed(BF16, ref, size, up_err, 64, 3)
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[5, 17] = bad
        out, got, w = g.moe_layer(y, router, w1, w2, 3, return_routing=True)
        assert torch.equal(got.cpu()[keep], ids.cpu()[keep]) and torch.equal(w.cpu()[keep], weights.cpu()[keep])
        assert ((out.cpu()[keep].double() - ref).abs() <= bound).all()
        assert out[5].isnan().all()


@pytest.mark.gpu
def test_hidden_values_beyond_fp16():
    """A hidden value of 10^5 is infinite in fp16, and so is what the down product makes of it; one of 60000 is not."""
    x = torch.full((2, 64), 1.0, dtype=FP16, device="cuda")
    x[1] = 0.75
    w1 = torch.zeros(1, 16, 64, dtype=FP16, device="cuda")
    w1[0, :8], w1[0, 8:] = 1000.0 / 64, 100.0 / 64             # gate 1000 and up 100, or 750 and 75
    w2 = torch.full((1, 64, 8), 1.0 / 16, dtype=FP16, device="cuda")
    out = g.moe_layer(x, torch.zeros(1, 64, dtype=FP16, device="cuda"), w1, w2, 1)
    assert (out[0] == math.inf).all()
    want = 8 * 750.0 * 75.0 / 16                                  # every number on the way is exact to 2^-11
    assert ((out[1].double() - want).abs() <= 4 * 2.0 ** -11 * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "mxfp4"])
def test_tokens_do_not_depend_on_their_company(fmt):
    """A token's routing is the same alone and in a batch."""
    x, router, w1, w2, *_ = make(40, 32, 512, 96, BF16, 8, fmt)
    _, ids, weights = g.moe_layer(x, router, w1, w2, 4, return_routing=True)
    for t in (0, 7, 29):
        for n in (1, 2, 9, 11):
            _, some, w = g.moe_layer(x[t:t + n].contiguous(), router, w1, w2, 4, return_routing=True)
            assert torch.equal(some, ids[t:t + n]) and torch.equal(w, weights[t:t + n])


@pytest.mark.gpu
def test_experts_behind_32_bits():
    """Expert rows beyond 2^32 bytes: the last of 40 experts of 128 MB is the one that is chosen."""
    E, H, I = 40, 8192, 4096
    gen = torch.Generator(device="cuda").manual_seed(1)
    w1 = torch.zeros(E, 2 * I, H, dtype=BF16, device="cuda")
    w2 = torch.zeros(E, H, I, dtype=BF16, device="cuda")
    w1[-1] = (torch.randn(2 * I, H, generator=gen, device="cuda") * H ** -0.5).to(BF16)
    w2[-1] = (torch.randn(H, I, generator=gen, device="cuda") * I ** -0.5).to(BF16)
    x = torch.randn(2, H, generator=gen, device="cuda").to(BF16)
    router = torch.zeros(E, H, dtype=BF16, device="cuda")
    bias = torch.zeros(E, device="cuda")
    bias[-1] = 5.0
    out, ids, weights = g.moe_layer(x, router, w1, w2, 1, bias=bias, return_routing=True)
    assert (ids == E - 1).all() and (weights == 1).all()
    ref, size, up_err = layer_ref(x, torch.zeros(2, 1, dtype=torch.int32), weights.cpu(), w1[-1:].cpu(), w2[-1:].cpu())
    assert ((out.double().cpu() - ref).abs() <= allowed(BF16, ref, size, up_err, I, 1)).all()


@pytest.mark.gpu
def test_streams_capture_and_workspace():
    x, router, w1, w2, *_ = make(10, 16, 256, 128, BF16, 31)
    x2 = make(10, 16, 256, 128, BF16, 32)[0]
    layer = lambda t, **kw: g.moe_layer(t, router, w1, w2, 4, **kw)  # noqa: E731
    want, want2 = layer(x), layer(x2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [layer(x, stream=side) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)
    # two captured layers on one workspace full of rubbish, replayed in turn
    ws = torch.full((g.moe_workspace_bytes(10, 16, 4, 256, 128),), 255, dtype=torch.uint8, device="cuda")
    static = x.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = layer(layer(static, workspace=ws), workspace=ws)
        graphs.append((graph, result))
    for source, first in ((x, want), (x2, want2)):
        static.copy_(source)
        expect = layer(first)
        for graph, result in graphs:
            graph.replay()
            assert torch.equal(result, expect)
    small = torch.empty(100, dtype=torch.uint8, device="cuda")
    with pytest.raises(g.GemmError, match="workspace"):
        layer(x, workspace=small)
    for out in (torch.empty(10, 256, device="cuda"), torch.empty(9, 256, dtype=BF16, device="cuda"), torch.empty(10, 256, dtype=BF16)):
        with pytest.raises(g.GemmError):
            layer(x, out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_quantised_experts_in_a_decode_step(fmt):
    """As a serving loop uses them together: 4-bit projections around a layer of 4-bit experts, against the same
    weights read back to bf16 and multiplied by the framework's 16-bit operators."""
    T, E, k, H, I = 6, 8, 2, 512, 256
    gen = torch.Generator().manual_seed(4)
    ts = 1.0 if fmt == "mxfp4" else 2.0 ** -6
    quant = lambda *s: g.quantize_mx((torch.randn(*s, generator=gen) * s[-1] ** -0.5).bfloat16().cuda(), fmt, tensor_scale=ts)  # noqa: E731
    proj, w1, w2 = quant(H, H), quant(E * 2 * I, H), quant(E * H, I)
    router = (torch.randn(E, H, generator=gen) * H ** -0.5).bfloat16().cuda()
    x = torch.randn(T, H, generator=gen).bfloat16().cuda()
    q = g.quantize_mx(x, fmt)
    hidden = g.gemm_mx(q, proj)
    out, ids, weights = g.moe_layer(hidden, router, w1, w2, k, return_routing=True)
    # the projection: the same values through the 16-bit GEMM (both sum the same exact products in fp32)
    other = g.gemm(g.dequantize_mx(q), g.dequantize_mx(proj))
    assert ((hidden.double() - other.double()).abs() <= 2.0 ** -7 * hidden.double().abs() + 1e-4).all()
    # the experts: the same values as 16-bit weights
    b1, b2 = g.dequantize_mx(w1).view(E, 2 * I, H), g.dequantize_mx(w2).view(E, H, I)
    same, ids16, w16 = g.moe_layer(hidden, router, b1, b2, k, return_routing=True)
    assert torch.equal(ids, ids16) and torch.equal(weights, w16)
    ref, size, up_err = layer_ref(hidden, ids.cpu(), weights.cpu(), b1.cpu(), b2.cpu())
    for o in (out, same):
        assert ((o.double().cpu() - ref).abs() <= allowed(BF16, ref, size, up_err, I, k)).all()

"""MxTensor as a Python object: copies, pickles, sizes and scales at the ends of their ranges."""
import copy
import io
import pickle

import pytest
import torch

import h100_gemm_b200 as g
from h100_gemm_b200 import api

FORMATS = ["mxfp4", "nvfp4"]


def saved_and_loaded(q):
    file = io.BytesIO()
    torch.save({"weight": q}, file)
    file.seek(0)
    return torch.load(file, weights_only=False)["weight"]


COPIES = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda q: pickle.loads(pickle.dumps(q)),
          "save": saved_and_loaded, "nested": lambda q: copy.deepcopy({"a": [q], "b": q})["b"]}


def cpu_matrix(rows, cols, fmt, one_allocation):
    if one_allocation:
        q = g.MxTensor._empty(rows, cols, fmt, 2.0 if fmt == "nvfp4" else 1.0, torch.device("cpu"))
    else:
        lib = api.library()
        q = g.MxTensor(torch.zeros(rows, lib.b200_mx_data_bytes(1, cols), dtype=torch.uint8),
                       torch.zeros(lib.b200_mx_scale_bytes({"mxfp4": 0, "nvfp4": 1}[fmt], rows, cols), dtype=torch.uint8),
                       rows, cols, fmt, 2.0 if fmt == "nvfp4" else 1.0)
    q.data.copy_(torch.randint(0, 256, q.data.shape, dtype=torch.uint8))
    q.scales.copy_(torch.randint(0, 127, q.scales.shape, dtype=torch.uint8))
    return q


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("one_allocation", [True, False])
@pytest.mark.parametrize("how", COPIES)
def test_copies_point_at_their_own_memory(how, one_allocation, fmt):
    q = cpu_matrix(70, 300, fmt, one_allocation)
    c = COPIES[how](q)
    assert (c.rows, c.cols, c.format, c.tensor_scale, c.device) == (q.rows, q.cols, q.format, q.tensor_scale, q.device)
    assert torch.equal(c.data, q.data) and torch.equal(c.scales, q.scales)
    for m in (q, c):
        assert m._data_ptr == m.data.data_ptr() and m._scales_ptr == m.scales.data_ptr()
        assert m._data_ptr % 16 == 0 and m._scales_ptr % 16 == 0
    if how == "copy":
        assert c._data_ptr == q._data_ptr                 # a shallow copy shares its tensors, as that of any object does
    else:
        before = q.data.clone()
        c.data.zero_()
        assert c._data_ptr != q._data_ptr and torch.equal(q.data, before)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("how", ["deepcopy", "pickle", "save"])
def test_copies_multiply_with_their_own_values(how, fmt):
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(200, 512, generator=gen).bfloat16().cuda()
    x = g.quantize_mx(torch.randn(5, 512, generator=gen).bfloat16().cuda(), fmt)
    q = g.quantize_mx(w, fmt)
    want = g.gemm_mx(x, q)
    c = COPIES[how](q)
    q.data.zero_()                                        # the original's memory is not what the copy reads
    assert not g.gemm_mx(x, q).any()
    del q
    assert torch.equal(g.gemm_mx(x, c), want)
    c.data.copy_(g.quantize_mx(-w, fmt).data)             # what is written into a copy is what it multiplies with
    assert torch.equal(g.gemm_mx(x, c), -want)
    assert torch.equal(g.dequantize_mx(c), g.dequantize_mx(g.quantize_mx(-w, fmt)))


def test_tensor_scales_that_fp32_cannot_hold():
    data, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2048, dtype=torch.uint8)
    for bad in (0.0, -1.0, 1e-50, 2.0 ** -130, 3.5e38, float("inf"), float("nan")):
        with pytest.raises(g.GemmError, match="tensor_scale"):
            g.MxTensor(data, scales, 4, 64, "nvfp4", bad)
    matrix = lambda ts: g.MxTensor(data, scales, 4, 64, "nvfp4", ts)  # noqa: E731
    # two legal scales whose product is not a number of fp32, or loses its bits
    for a, b, alpha in ((2.0 ** 64, 2.0 ** 64, 1.0), (1e30, 1e30, 1.0), (2.0 ** 64, 1.0, 2.0 ** 64), (1e-25, 1e-25, 1.0),
                        (1e-20, 1e-20, 0.3), (2.0 ** 64, 2.0 ** 64, -1.0)):
        with pytest.raises(g.GemmError, match="outside fp32's range"):
            g.gemm_mx(matrix(a), matrix(b), alpha=alpha)
    # the same undone by alpha, powers of two that are exact, and what an alpha means by itself: refused for the device alone
    for a, b, alpha in ((2.0 ** 64, 2.0 ** 64, 2.0 ** -100), (2.0 ** -64, 2.0 ** -64, 1.0), (2.0 ** 64, 2.0 ** 64, 0.0),
                        (1e-25, 1e-25, 1e20), (1.0, 1.0, float("inf")), (1.0, 1.0, float("nan"))):
        with pytest.raises(g.GemmError, match="CUDA tensor"):
            g.gemm_mx(matrix(a), matrix(b), alpha=alpha)


def test_tensor_scales_of_expert_weights_are_checked():
    p = 4096
    call = lambda fmt, t1, t2: api.library().b200_moe_layer(0, 2, 8, 2, 64, 32, p, p, None, fmt, p, p, t1, p, p, t2, 1, p, None, None,  # noqa: E731
                                                            None, 0, None)
    for bad in (0.0, -1.0, float("inf"), float("nan"), -float("inf")):
        assert call(1, bad, 1.0) == call(1, 1.0, bad) == api.STATUS_INVALID_ARG
    assert call(0, 2.0, 1.0) == call(0, 1.0, 0.5) == api.STATUS_INVALID_ARG
    for good in ((0, 1.0, 1.0), (1, 0.37, 3e38)):                    # past the checks: no workspace
        assert call(*good) == api.STATUS_WORKSPACE


@pytest.mark.gpu
def test_products_under_far_tensor_scales():
    """Scales of 2^64 and 2^-64 on both sides, brought back by alpha: the same bits, and zeros stay zeros."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(300, 512, generator=gen)
    x[3] = 0
    x = x.bfloat16().cuda()
    base = g.quantize_mx(x, "nvfp4")
    want = g.gemm_mx(base, base)
    assert not want[3].any() and want.isfinite().all()
    for e in (64, -64):
        q = g.quantize_mx((x.double() * 2.0 ** e).bfloat16(), "nvfp4", tensor_scale=2.0 ** e)
        assert torch.equal(g.gemm_mx(q, q, alpha=2.0 ** (-2 * e)), want)
        assert torch.equal(g.gemm_mx(q, base, alpha=2.0 ** -e), want)
    q = g.quantize_mx((x.double() * 2.0 ** -50).bfloat16(), "nvfp4", tensor_scale=2.0 ** -50)
    assert torch.equal(g.gemm_mx(q, q).double(), want.double() * 2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("e1,e2", [(100, 112), (-100, -100), (-124, -100)])
def test_experts_under_far_tensor_scales(e1, e2):
    """NVFP4 experts whose tensor scales are far from 1, undone by the tokens (gate and up) or seen in the result."""
    T, E, k, H, I = 3, 4, 2, 64, 48
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(T, H, generator=gen).bfloat16().cuda()
    router = torch.zeros(E, H, dtype=torch.bfloat16, device="cuda")
    w1 = g.quantize_mx(torch.randn(E * 2 * I, H, generator=gen).bfloat16().cuda(), "nvfp4")
    w2 = g.quantize_mx(torch.randn(E * H, I, generator=gen).bfloat16().cuda(), "nvfp4")
    want = g.moe_layer(x, router, w1, w2, k)
    far = lambda q, e: g.MxTensor(q.data, q.scales, q.rows, q.cols, "nvfp4", 2.0 ** e)  # noqa: E731
    undone = (x.double() * 2.0 ** -e1).bfloat16()
    assert torch.equal(g.moe_layer(undone, router, far(w1, e1), w2, k), want)
    assert torch.equal(g.moe_layer(x, router, w1, far(w2, e2), k).double(), want.double() * 2.0 ** e2)


def test_sizes_beyond_32_bits_are_refused():
    """The C ABI's sizes are 32-bit: 2^32 + 5 rows would arrive as 5."""
    BF16 = torch.bfloat16
    big = 2 ** 32 + 8
    meta = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    for x in (meta(big, 1), meta(1, big), meta(2 ** 31, 2)):
        for call in (g.quantize_mx, g.quantize_mx_both, lambda t: g.quantize_mx(t, transpose=True)):
            with pytest.raises(g.GemmError, match="rows and columns"):
                call(x)
    with pytest.raises(g.GemmError, match="rows and columns"):
        g.MxTensor(meta(big * 16, dtype=torch.uint8), meta(1, dtype=torch.uint8), big, 32)
    for H, I in ((big, 8), (8, big), (2 ** 20 + 8, 8)):
        with pytest.raises(g.GemmError, match="hidden and inner"):
            g.moe_layer(meta(1, H), meta(2, H), meta(2, 2 * I, H), meta(2, H, I), 1)
        assert g.moe_workspace_bytes(1, 2, 1, H, I) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 67])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_read_back_are_rounded_once(dtype, cols):
    """Tensor scales that put code * scale next to the middle between two 16-bit numbers, nearer than fp32 can tell."""
    half = torch.finfo(dtype).eps / 2
    code = torch.full((1, (cols + 1) // 2), 5 | 13 << 4, dtype=torch.uint8)           # 3 and -3
    block = torch.full((1, -(-cols // 16)), 0x38, dtype=torch.uint8)                   # 1
    sides = set()
    for k in range(40):
        middle = 1 + half * (2 * k + 1)
        ts = torch.tensor(middle / 3, dtype=torch.float64).float().double().item()
        q = g.MxTensor.from_parts(code.cuda(), block.cuda(), cols, "nvfp4", ts)
        value = 3 * ts                                                               # exact in 64 bits
        sides.add((value > middle) - (value < middle))
        want = torch.tensor(1 + 2 * half * (k + (value > middle) + (value == middle) * (k % 2)), dtype=torch.float64)
        got = g.dequantize_mx(q, dtype).double().cpu()[0]
        assert (got[0::2] == want).all() and (got[1::2] == -want).all(), (k, got[:2], want)
    assert {-1, 1} <= sides

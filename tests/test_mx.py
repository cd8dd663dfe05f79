"""Microscaled 4-bit operators: quantisation, its inverse and the product, against their definition in
64 bits (numpy, written from the formulas in include/b200_gemm.h)."""
import math

import numpy as np
import pytest
import torch

import h100_gemm_b200 as g
from h100_gemm_b200 import api

FORMATS = ["mxfp4", "nvfp4"]
BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAG = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# every non-negative e4m3 number, by byte
E4M3 = np.array([(b & 7) * 2.0 ** -9 if b < 8 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(127)])


def nearest(values, table):
    """Index of the nearest table entry; ties to the even index; beyond the end the last one."""
    mids = (table[:-1] + table[1:]) / 2
    low = np.searchsorted(mids, values, side="left")     # a value on a border stays below it
    high = np.searchsorted(mids, values, side="right")   # ... or goes above it
    return np.where(low % 2 == 0, low, high)


def quantise_ref(x, fmt, ts=1.0):
    """x [R, C] float64 -> codes [R, C], scale bytes [R, blocks], values [R, C]."""
    R, C = x.shape
    blk = BLOCK[fmt]
    y = np.zeros((R, -(-C // blk) * blk))
    y[:, :C] = x
    y = y.reshape(R, -1, blk)
    amax = np.abs(y).max(axis=2)
    bad = ~np.isfinite(amax)
    safe = np.where(bad | (amax == 0), 1.0, amax)
    if fmt == "mxfp4":
        e = np.where(amax == 0, -127, np.clip(np.frexp(safe)[1] - 3, -127, 125))
        byte, scale = np.where(bad, 255, e + 127), np.ldexp(1.0, e)
    else:
        byte = nearest(np.where(amax == 0, 0.0, safe) / (6.0 * ts), E4M3)
        scale = E4M3[byte] * ts
        byte = np.where(bad, 127, byte)
    with np.errstate(invalid="ignore"):
        ratio = np.where(scale[:, :, None] > 0, np.abs(y) / np.where(scale > 0, scale, 1.0)[:, :, None], 0.0)
    ratio = np.where(bad[:, :, None], 0.0, ratio)
    code = nearest(ratio, MAG)
    value = MAG[code] * scale[:, :, None] * np.where(y < 0, -1.0, 1.0)
    value = np.where(bad[:, :, None], np.nan, value)
    code = np.where(bad[:, :, None], 0, code)
    return code.reshape(R, -1)[:, :C], byte.astype(np.uint8), value.reshape(R, -1)[:, :C]


def to64(t):
    return t.double().cpu().numpy()


def activations(rows, cols, dtype, seed, special=False):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen)
    x *= torch.exp2(torch.randint(-12, 9, (rows, 1), generator=gen).float())
    if special:
        x[0] = 0.0
        flat = x.view(-1)
        n = flat.numel()
        # borders between codes and between scales, the types' smallest and largest numbers, infinities, NaN
        table = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 7.0, 2.0 ** -14, 2.0 ** -24, 65504.0, -0.0]
        for i, v in enumerate(table * 3):
            flat[(i * 37 + 11) % n] = v
        flat[n // 2], flat[n // 3], flat[n - 1] = math.inf, math.nan, -math.inf
        if dtype == torch.bfloat16:
            for i, v in enumerate([3.3e38, -3.3e38, 2.0 ** -126, 2.0 ** -133, 2.0 ** -130 * 1.5]):
                flat[(i * 53 + 200) % n] = v
    return x.to(dtype)


def random_mx(rows, cols, fmt, seed, scale_low, scale_high, tensor_scale=1.0):
    """Random codes and scale bytes in [scale_low, scale_high], and the values they stand for."""
    rng = np.random.Generator(np.random.Philox(seed))
    blocks = -(-cols // BLOCK[fmt])
    code = rng.integers(0, 16, (rows, -(-cols // 2) * 2), dtype=np.uint8)
    code[:, cols:] = 0
    byte = rng.integers(scale_low, scale_high + 1, (rows, blocks)).astype(np.uint8)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    m = g.MxTensor.from_parts(torch.from_numpy(packed).cuda(), torch.from_numpy(byte).cuda(), cols, fmt, tensor_scale)
    scale = np.ldexp(1.0, byte.astype(int) - 127) if fmt == "mxfp4" else E4M3[byte]
    value = MAG[code & 7] * np.where(code >= 8, -1.0, 1.0)
    value = value[:, :cols] * np.repeat(scale, BLOCK[fmt], axis=1)[:, :cols] * tensor_scale
    return m, value


def check_quantised(q, x, fmt, ts=1.0):
    code, byte, value = quantise_ref(x, fmt, ts)
    got_code, got_byte = (t.cpu().numpy() for t in q.to_parts())
    np.testing.assert_array_equal(got_byte, byte)
    C = x.shape[1]
    unpacked = np.stack([got_code & 15, got_code >> 4], axis=2).reshape(x.shape[0], -1)
    np.testing.assert_array_equal(unpacked[:, :C] & 7, code)
    sign = unpacked[:, :C] >= 8
    np.testing.assert_array_equal(sign[code > 0], (x < 0)[code > 0])
    assert not unpacked[:, C:].any() and not q.data[:, (C + 1) // 2:].any()  # what a row has beyond its columns is zero
    return value


def check_padding(q):
    """The scale bytes of padding rows and columns are zero."""
    clean = g.MxTensor.from_parts(*q.to_parts(), q.cols, q.format, q.tensor_scale)
    assert torch.equal(clean.scales, q.scales)


# --------------------------------------------------------------------------------------- no GPU
def cpu_mx(rows, cols, fmt="mxfp4", ts=1.0):
    lib = api.library()
    return g.MxTensor(torch.zeros(rows, lib.b200_mx_data_bytes(1, cols), dtype=torch.uint8),
                      torch.zeros(lib.b200_mx_scale_bytes({"mxfp4": 0, "nvfp4": 1}[fmt], rows, cols), dtype=torch.uint8),
                      rows, cols, fmt, ts)


def test_sizes():
    lib = api.library()
    assert lib.b200_mx_data_bytes(3, 65) == 3 * 48       # 33 bytes of codes, rows on 16 bytes
    assert lib.b200_mx_data_bytes(1, 1) == 16
    assert lib.b200_mx_scale_bytes(0, 1, 1) == 1024 and lib.b200_mx_scale_bytes(1, 1, 1) == 2048
    assert lib.b200_mx_scale_bytes(0, 129, 257) == 4 * 1024
    assert lib.b200_mx_scale_bytes(0, 1 << 20, 1 << 20) == (1 << 40) // 32  # offsets beyond 32 bits
    assert lib.b200_mx_scale_bytes(2, 1, 1) == 0 and lib.b200_mx_data_bytes(0, 4) == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 33), (129, 300), (128, 256)])
def test_parts_round_trip(fmt, rows, cols):
    rng = np.random.Generator(np.random.Philox(1))
    codes = torch.from_numpy(rng.integers(0, 256, (rows, (cols + 1) // 2), dtype=np.uint8))
    if cols % 2:
        codes[:, -1] &= 15
    scales = torch.from_numpy(rng.integers(0, 127, (rows, -(-cols // BLOCK[fmt])), dtype=np.uint8))
    m = g.MxTensor.from_parts(codes, scales, cols, fmt)
    back = m.to_parts()
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)
    # the documented place of every scale byte
    groups = 256 // BLOCK[fmt] // 4
    col_tiles = -(-cols // 256)
    for r in {0, rows // 2, rows - 1}:
        for b in range(scales.shape[1]):
            at = ((r // 128) * col_tiles * groups + b // 4) * 512 + (r % 32) * 16 + r % 128 // 32 * 4 + b % 4
            assert m.scales[at] == scales[r, b]


def test_refusals_without_a_device():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: g.quantize_mx(x), lambda: g.quantize_mx_both(x), lambda: g.dequantize_mx(cpu_mx(4, 64)),
                 lambda: g.gemm_mx(cpu_mx(4, 64), cpu_mx(4, 64))):
        with pytest.raises(g.GemmError, match="CUDA tensor"):
            call()
    with pytest.raises(g.GemmError, match="bfloat16 or float16"):
        g.quantize_mx(x.float())
    with pytest.raises(g.GemmError, match="format"):
        g.quantize_mx(x, "int4")
    for bad in (x[0], x[:0], x[:, :0], x.t()):
        with pytest.raises(g.GemmError):
            g.quantize_mx(bad)
    with pytest.raises(g.GemmError, match="overlap"):
        g.quantize_mx(x[:1].expand(4, 64))
    with pytest.raises(g.GemmError, match="disagree on K"):
        g.gemm_mx(cpu_mx(4, 64), cpu_mx(4, 32))
    with pytest.raises(g.GemmError, match="mxfp4"):
        g.gemm_mx(cpu_mx(4, 64), cpu_mx(4, 64, "nvfp4"))
    with pytest.raises(g.GemmError, match="tensor scale"):
        cpu_mx(4, 64, "mxfp4", 2.0)
    with pytest.raises(g.GemmError):
        cpu_mx(4, 64, "nvfp4", math.inf)
    for call in (lambda: g.gemm_mx(x, cpu_mx(4, 64)), lambda: g.gemm_mx(cpu_mx(4, 64), x), lambda: g.dequantize_mx(x)):
        with pytest.raises(g.GemmError, match="MxTensor"):
            call()
    good = cpu_mx(4, 64)
    with pytest.raises(g.GemmError, match="bytes"):
        g.MxTensor(good.data, good.scales, 5, 64)
    with pytest.raises(g.GemmError, match="contiguous uint8"):
        g.MxTensor(good.data.float(), good.scales, 4, 64)


def test_refusals_of_the_c_abi():
    """Arguments are refused before any device is asked for."""
    lib = api.library()
    p = 4096  # a pointer that is never followed
    ok = dict(fmt=0, f16=0, rows=4, cols=64, x=p, ld=64, ts=1.0, d=p, s=p, dt=None, st=None)

    def quant(**kw):
        a = {**ok, **kw}
        return lib.b200_mx_quantize(a["fmt"], a["f16"], a["rows"], a["cols"], a["x"], a["ld"], a["ts"], a["d"], a["s"],
                                    a["dt"], a["st"], None)

    for kw in (dict(fmt=2), dict(rows=0), dict(cols=-1), dict(x=None), dict(ld=63), dict(d=None), dict(d=p + 8),
               dict(s=p + 4), dict(dt=p), dict(d=None, s=None), dict(x=p + 1), dict(ts=2.0), dict(fmt=1, ts=3.0),
               dict(fmt=1, ts=0.0), dict(fmt=1, ts=-1.0), dict(fmt=1, ts=math.nan), dict(fmt=1, ts=2.0 ** 65)):
        assert quant(**kw) == api.STATUS_INVALID_ARG, kw
    for args in ((2, 0, 4, 4, 64, p, p, p, p, p), (0, 0, 0, 4, 64, p, p, p, p, p), (0, 0, 4, 4, 0, p, p, p, p, p),
                 (0, 0, 4, 4, 64, None, p, p, p, p), (0, 0, 4, 4, 64, p, p + 1, p, p, p), (0, 0, 4, 4, 64, p, p, p, p, p + 1), (0, 0, 2 ** 31 - 1, 4, 64, p, p, p, p, p)):
        assert lib.b200_gemm_mx(*args, 1.0, 0.0, None) == api.STATUS_INVALID_ARG, args
    for args in ((3, 0, 4, 64, p, p, 1.0, p, 64), (0, 0, 4, 64, p + 1, p, 1.0, p, 64), (0, 0, 4, 64, p, p, 1.0, p, 63),
                 (0, 0, 4, 64, p, p, 2.0, p, 64), (1, 0, 4, 64, p, p, 0.0, p, 64), (1, 0, 4, 64, p, p, math.nan, p, 64),
                 (1, 0, 4, 64, p, p, math.inf, p, 64)):
        assert lib.b200_mx_dequantize(*args, None) == api.STATUS_INVALID_ARG, args


# --------------------------------------------------------------------------------------- quantisation
SHAPES = [(1, 1), (1, 32), (3, 17), (16, 256), (127, 129), (128, 128), (129, 513), (300, 1000), (33, 4104)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantise_is_exact(rows, cols, fmt, dtype):
    x = activations(rows, cols, dtype, rows * 7 + cols, special=rows * cols > 1000).cuda()
    ref = to64(x)
    q, qt = g.quantize_mx_both(x, fmt)
    values = check_quantised(q, ref, fmt)
    values_t = check_quantised(qt, ref.T, fmt)
    check_padding(q)
    check_padding(qt)
    one, one_t = g.quantize_mx(x, fmt), g.quantize_mx(x, fmt, transpose=True)
    for a, b in ((q, one), (qt, one_t)):
        assert torch.equal(a.data, b.data) and torch.equal(a.scales, b.scales)
    # the values, rounded to the type once
    for m, v in ((q, values), (qt, values_t)):
        got = g.dequantize_mx(m, dtype)
        with np.errstate(over="ignore"):
            want = torch.from_numpy(v).to(torch.float32).to(dtype)  # (the values are exact in fp32)
        np.testing.assert_array_equal(to64(got), to64(want))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_every_bf16_number(fmt):
    """Every finite bf16 number against every scale its block can have: one block, the number first,
    a power of two times 1..1.875 as the largest magnitude."""
    bits = torch.arange(0, 0x7F80, dtype=torch.int32)
    rows = []
    for top in (1.0, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875, 6.0 * 448, 6.0 * 500, 2.0 ** -9 * 6, 2.0 ** -10 * 6, 2.0 ** -11 * 6):
        x = torch.zeros(0x7F80, BLOCK[fmt], dtype=torch.bfloat16)
        x[:, 0] = bits.to(torch.int16).view(torch.bfloat16)
        x[:, 1] = -top
        rows.append(x)
    x = torch.cat(rows).cuda()
    check_quantised(g.quantize_mx(x, fmt), to64(x), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-64, -30, -8, 3, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise_with_a_tensor_scale(dtype, exponent):
    ts = 2.0 ** exponent
    x = activations(70, 200, dtype, 5).cuda()
    q, qt = g.quantize_mx_both(x, "nvfp4", tensor_scale=ts)
    check_quantised(q, to64(x), "nvfp4", ts)
    check_quantised(qt, to64(x).T, "nvfp4", ts)
    assert q.tensor_scale == ts


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_strided_and_misaligned(fmt):
    base = activations(90, 800, torch.bfloat16, 9).cuda()
    for x in (base[:, 8:360], base[:, 1:300], base[::3, 3:64], base[5:6, 7:400], base.view(-1)[1:1 + 40 * 100].view(40, 100)):
        q, qt = g.quantize_mx_both(x, fmt)
        check_quantised(q, to64(x), fmt)
        check_quantised(qt, to64(x).T, fmt)
        out = torch.full((x.shape[0], x.shape[1] + 13), 7.0, dtype=torch.bfloat16, device="cuda")
        g.dequantize_mx(q, out=out[:, 5:5 + x.shape[1]])
        np.testing.assert_array_equal(to64(out[:, 5:5 + x.shape[1]]), to64(g.dequantize_mx(q)))
        assert (out[:, :5] == 7).all() and (out[:, 5 + x.shape[1]:] == 7).all()  # neighbours left as they were


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_dequantise_every_scale(fmt):
    """All 256 codes of a byte against every scale byte, NaN included."""
    top = 256 if fmt == "mxfp4" else 128
    codes = torch.arange(256, dtype=torch.uint8).repeat(top, 1)
    blocks = 512 // BLOCK[fmt]
    scales = torch.arange(top, dtype=torch.int32).to(torch.uint8)[:, None].repeat(1, blocks)
    m = g.MxTensor.from_parts(codes.cuda(), scales.cuda(), 512, fmt, 1.0 if fmt == "mxfp4" else 0.25)
    c = np.stack([np.arange(256) & 15, np.arange(256) >> 4], axis=1).reshape(-1)
    value = (MAG[c & 7] * np.where(c >= 8, -1.0, 1.0))[None, :]
    if fmt == "mxfp4":
        value = value * np.ldexp(1.0, np.arange(256) - 127)[:, None]
        value[255] = np.nan
    else:
        value = value * np.append(E4M3, np.nan)[:, None] * 0.25
    for dtype in (torch.bfloat16, torch.float16):
        with np.errstate(over="ignore"):
            # 4 significant bits at most times 2: exact in 64 bits; one rounding to the type (through fp32,
            # whose 24 bits hold 6 exactly down to its own subnormals and beyond its largest become infinite alike)
            want = torch.from_numpy(value).float().to(dtype)
        np.testing.assert_array_equal(to64(g.dequantize_mx(m, dtype)), to64(want))


# --------------------------------------------------------------------------------------- product
def product_bound(a, b, ref, dtype):
    """|C - ref| allowed: half a step of the output type, plus fp32 accumulation. Products of codes are exact; every
    MMA adds K = 64 of them to the accumulator with an error of at most 2^-22 of the magnitudes involved
    (fp32 with one guard bit lost in the alignment), and joining up to 8 partial sums adds 8 roundings."""
    K = a.shape[1]
    return torch.finfo(dtype).eps / 2 * np.abs(ref) + (K / 64 + 9) * 2.0 ** -22 * (np.abs(a) @ np.abs(b).T) + \
        torch.finfo(dtype).tiny * torch.finfo(dtype).eps


PRODUCTS = [(1, 128, 256), (1, 4096, 4096), (2, 130, 64), (16, 1000, 520), (17, 300, 2048), (32, 128, 8192), (33, 1024, 1024),
            (64, 257, 3000), (65, 640, 512), (128, 128, 16384), (128, 2048, 768), (129, 128, 256), (200, 100, 1000),
            (257, 300, 513), (128, 1, 31), (300, 3, 33), (1, 1, 1), (512, 1024, 2048), (1000, 1544, 700), (700, 999, 4100)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(M, N, K, fmt):
    low, high = (120, 129) if fmt == "mxfp4" else (0, 126)
    ts = (1.0, 1.0) if fmt == "mxfp4" else (2.0 ** -6, 0.37)
    a, av = random_mx(M, K, fmt, M + N, low, high, ts[0])
    b, bv = random_mx(N, K, fmt, K + 3, low, high, ts[1])
    ref = av @ bv.T
    for dtype in (torch.bfloat16, torch.float16):
        alpha = 1.0 if dtype == torch.bfloat16 else 2.0 ** -12  # (inside fp16's range)
        out = torch.full((M, N), math.nan, dtype=dtype, device="cuda")
        assert g.gemm_mx(a, b, out=out, alpha=alpha) is out
        # (alpha times the tensor scales is rounded to fp32, and its product with the sum once more)
        bound = product_bound(av * alpha, bv, ref * alpha, dtype) + 2.0 ** -23 * np.abs(ref * alpha)
        bad = ~(np.abs(to64(out) - ref * alpha) <= bound)
        assert not bad.any(), f"{bad.sum()} of {bad.size} outside, first {np.argwhere(bad)[:4].tolist()}"
    assert g.device_status()[0] == api.STATUS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 16, 48, 128, 300])
@pytest.mark.parametrize("fmt", FORMATS)
def test_product_of_small_integers_is_exact(fmt, M):
    """Scales of one: sums of multiples of 1/4 stay exact in fp32, so the output is the nearest bf16 number."""
    one = 127 if fmt == "mxfp4" else 0x38
    a, av = random_mx(M, 1500, fmt, 1, one, one)
    b, bv = random_mx(260, 1500, fmt, 2, one, one)
    ref = av @ bv.T * 0.5 + 3.0
    got = g.gemm_mx(a, b, alpha=0.5, beta=3.0)
    np.testing.assert_array_equal(to64(got), to64(torch.from_numpy(ref).float().bfloat16()))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [3, 200])
def test_product_scales_by_block(fmt, M):
    """One block of ones at a time, each under a scale of its own: every scale reaches its block."""
    K = 1024
    blocks = K // BLOCK[fmt]
    low = 100 if fmt == "mxfp4" else 8
    codes = torch.full((M, K // 2), 0x22, dtype=torch.uint8, device="cuda")  # all ones
    sa = (low + torch.arange(M)[:, None] % 5 + torch.arange(blocks)[None, :] % 7).to(torch.uint8).cuda()
    a = g.MxTensor.from_parts(codes, sa, K, fmt)
    cb = torch.zeros(blocks, K // 2, dtype=torch.uint8, device="cuda")
    for i in range(blocks):
        cb[i, i * BLOCK[fmt] // 2:(i + 1) * BLOCK[fmt] // 2] = 0x22
    sb = (low + 3 + torch.arange(blocks)[:, None] % 3 + torch.zeros(1, blocks)).to(torch.uint8).cuda()
    b = g.MxTensor.from_parts(cb, sb, K, fmt)
    val = (lambda t: np.ldexp(1.0, t.cpu().numpy().astype(int) - 127)) if fmt == "mxfp4" else (lambda t: E4M3[t.cpu().numpy()])
    ref = BLOCK[fmt] * val(sa) * np.diag(val(sb))[None, :]
    np.testing.assert_array_equal(to64(g.gemm_mx(a, b)), to64(torch.from_numpy(ref).float().bfloat16()))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [5, 200])
def test_product_keeps_nan_to_its_row(fmt, M):
    x = activations(M, 512, torch.bfloat16, 3).cuda()
    w = activations(300, 512, torch.bfloat16, 4).cuda()
    x[2, 100], w[7, 3] = math.inf, math.nan
    out = g.gemm_mx(g.quantize_mx(x, fmt), g.quantize_mx(w, fmt))
    want = torch.zeros(M, 300, dtype=torch.bool, device="cuda")
    want[2], want[:, 7] = True, True
    assert torch.equal(out.isnan(), want)


@pytest.mark.gpu
def test_product_output_refusals_and_neighbours():
    a, _ = random_mx(40, 320, "mxfp4", 1, 120, 128)
    b, _ = random_mx(72, 320, "mxfp4", 2, 120, 128)
    for out in (torch.empty(72, 40, dtype=torch.bfloat16, device="cuda"), torch.empty(40, 72, device="cuda"),
                torch.empty(40, 80, dtype=torch.bfloat16, device="cuda")[:, :72], torch.empty(40, 72, dtype=torch.bfloat16)):
        with pytest.raises(g.GemmError):
            g.gemm_mx(a, b, out=out)
    pool = torch.full((41 * 72 + 1,), 5.0, dtype=torch.bfloat16, device="cuda")
    out = pool[1:1 + 40 * 72].view(40, 72)  # not on 16 bytes
    g.gemm_mx(a, b, out=out)
    assert torch.equal(out, g.gemm_mx(a, b)) and pool[0] == 5 and (pool[1 + 40 * 72:] == 5).all()


# --------------------------------------------------------------------------------------- together
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(64, 136, 200), (300, 257, 514)])
def test_linear_layer_and_its_gradients(M, N, K, dtype, fmt):
    """y = q(x) q(w)^T, dx = q(dy) q(w^T)^T, dw = q(dy^T) q(x^T)^T: the formulas in 64 bits on the quantised operands,
    and against differences of the layer's own loss sum(dy * y), in which the same operands are quantised."""
    gen = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=gen).to(dtype).cuda()
    w = (torch.randn(N, K, generator=gen) * 0.05).to(dtype).cuda()
    dy = (torch.randn(M, N, generator=gen) * 2.0 ** -9).to(dtype).cuda()
    ws, ds = (2.0 ** -7, 2.0 ** -10) if fmt == "nvfp4" else (1.0, 1.0)
    xr, xc = g.quantize_mx_both(x, fmt)
    wr, wc = g.quantize_mx_both(w, fmt, tensor_scale=ws)
    dr, dc = g.quantize_mx_both(dy, fmt, tensor_scale=ds)
    got = g.gemm_mx(xr, wr, dtype=dtype), g.gemm_mx(dr, wc, dtype=dtype), g.gemm_mx(dc, xc, dtype=dtype)
    q = {}
    for name, t, s in (("x", x, 1.0), ("w", w, ws), ("dy", dy, ds)):
        q[name], q[name + "t"] = quantise_ref(to64(t), fmt, s)[2], quantise_ref(to64(t).T, fmt, s)[2]
    for out, a, b in ((got[0], q["x"], q["w"]), (got[1], q["dy"], q["wt"]), (got[2], q["dyt"], q["xt"])):
        ref = a @ b.T
        assert (np.abs(to64(out) - ref) <= product_bound(a, b, ref, dtype) + 2.0 ** -23 * np.abs(ref)).all()
    # Differences: the loss is linear in each operand, so a step of any length gives its derivative exactly;
    # along a direction v, sum(dy * (q(x) + h v) w^T) changes by h sum(v * dx). dx here is from operands
    # quantised along N, so the comparison holds for that product's own operands.
    v = np.random.Generator(np.random.Philox(1)).standard_normal((M, K))
    loss = lambda xx: (q["dy"] * (xx @ q["wt"])).sum()  # noqa: E731
    h = 0.5
    diff = (loss(q["x"] + h * v) - loss(q["x"] - h * v)) / (2 * h)
    ref = q["dy"] @ q["wt"].T
    slack = (product_bound(q["dy"], q["wt"], ref, dtype) + 2.0 ** -23 * np.abs(ref)) * np.abs(v)
    assert abs((to64(got[1]) * v).sum() - diff) <= slack.sum() + 1e-9


@pytest.mark.gpu
def test_streams_capture_and_repeat():
    """Another stream than the current one, and a captured pass replayed on new inputs, give the same bits."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(20, 3000, generator=gen).bfloat16().cuda()
    x2 = torch.randn(20, 3000, generator=gen).bfloat16().cuda()
    w = g.quantize_mx((torch.randn(500, 3000, generator=gen) * 0.02).bfloat16().cuda(), "nvfp4", tensor_scale=2.0 ** -8)
    layer = lambda t, stream=None: g.gemm_mx(g.quantize_mx(t, "nvfp4", stream=stream), w, stream=stream)  # noqa: E731
    want, want2 = layer(x), layer(x2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [layer(x, side) for _ in range(3)] + [layer(x, side.cuda_stream)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)
    static = x.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = layer(static)
        graphs.append((graph, result))
    for source, expect in ((x, want), (x2, want2), (x, want)):
        static.copy_(source)
        for graph, _ in graphs:
            graph.replay()
        assert all(torch.equal(result, expect) for _, result in graphs)
    assert g.device_status()[0] == api.STATUS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(65, 8200, 1100), (256, 18944, 512), (257, 19000, 300), (300, 256, 9000), (2100, 4800, 1030), (3000, 2999, 257),
                                   (16, 40000, 300), (64, 38000, 700), (1, 60000, 256), (4097, 513, 2048), (600, 600, 24000), (777, 5008, 1100), (777, 5003, 1100), (900, 4610, 600), (300, 40001, 300)])
def test_product_many_tiles(M, N, K, fmt):
    """More tiles than the device takes at a time, ragged ends, long contractions shared by a cluster."""
    low, high = (125, 129) if fmt == "mxfp4" else (0x28, 0x40)
    a, av = random_mx(M, K, fmt, M + N, low, high)
    b, bv = random_mx(N, K, fmt, K + 3, low, high)
    out = torch.full((M, N), math.nan, dtype=torch.bfloat16, device="cuda")
    g.gemm_mx(a, b, out=out)
    bad = 0
    bv32 = torch.from_numpy(bv).cuda()
    for r in range(0, M, 512):  # (in slices: the reference is 64-bit)
        rows = torch.from_numpy(av[r:r + 512]).cuda()
        ref = rows @ bv32.T
        bound = 2.0 ** -8 * ref.abs() + (K / 64 + 9) * 2.0 ** -22 * (rows.abs() @ bv32.abs().T)
        bad += int((~((out[r:r + 512].double() - ref).abs() <= bound)).sum())
    assert bad == 0, f"{bad} of {M * N} outside"
    assert torch.equal(out, g.gemm_mx(a, b))
    assert g.device_status()[0] == api.STATUS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise_borders_of_every_scale(fmt, dtype):
    """Every border between two codes, exactly and one step of the type to either side, under every scale a block
    can have: a block's largest magnitude decides the scale, the borders of that scale fill the rest."""
    blk = BLOCK[fmt]
    if fmt == "mxfp4":
        scales = np.ldexp(1.0, np.arange(-20, 13))
        tops = np.array([4.0, 6.0, 7.0])
    else:
        scales = E4M3[1:]
        tops = np.array([6.0])
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for s in scales:
        for top in tops:
            base = torch.from_numpy(np.concatenate([[top * s], borders * s])).to(dtype)
            bits = base.view(torch.int16).int()
            for step in (-1, 0, 1):
                moved = bits.clone()
                moved[1:] += step
                row = torch.zeros(blk, dtype=dtype)
                row[:8] = moved.to(torch.int16).view(dtype)
                rows.append(row)
    x = torch.stack(rows).cuda()
    x = torch.cat([x, -x])
    q, qt = g.quantize_mx_both(x, fmt)
    check_quantised(q, to64(x), fmt)
    check_quantised(qt, to64(x).T, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", range(8))
def test_quantise_rows_at_every_offset(offset, dtype, fmt):
    """Rows that start anywhere between two 16-byte boundaries, odd row distances, tiles cut at either end; what lies
    around the matrix is NaN and stays where it is."""
    for rows, cols, ld in ((130, 259, 301), (3, 1, 9), (129, 127, 128), (40, 131, 137), (2, 300, 300)):
        pool = torch.full((offset + rows * ld + 16,), math.nan, dtype=dtype, device="cuda")
        x = pool[offset:offset + rows * ld].view(rows, ld)[:, :cols]
        x.copy_(activations(rows, cols, dtype, rows + offset).cuda())
        q, qt = g.quantize_mx_both(x, fmt)
        values = check_quantised(q, to64(x), fmt)
        check_quantised(qt, to64(x).T, fmt)
        one = g.quantize_mx(x, fmt)
        assert torch.equal(one.data, q.data) and torch.equal(one.scales, q.scales)
        back = pool.clone()
        g.dequantize_mx(q, out=back[offset:offset + rows * ld].view(rows, ld)[:, :cols])
        inside = torch.zeros_like(pool, dtype=torch.bool)
        inside[offset:offset + rows * ld].view(rows, ld)[:, :cols] = True
        assert back[~inside].isnan().all()
        np.testing.assert_array_equal(to64(back[inside]), to64(torch.from_numpy(values).float().to(dtype)).reshape(-1))


@pytest.mark.gpu
def test_between_products_with_short_rings():
    """A 16-bit product of two stages leaves an SM room for a 4-bit one beside it: both need tensor memory, and each
    begins while the other still runs. Captured, so that nothing but the kernels keeps them in order."""
    gen = torch.Generator().manual_seed(8)
    a = torch.randn(700, 512, generator=gen).bfloat16().cuda()
    b = (torch.randn(512, 512, generator=gen) * 512 ** -0.5).bfloat16().cuda()
    cfg = api.GemmConfig(block_n=256, cluster_m=1, stages=2)
    w, small = g.quantize_mx(b), g.quantize_mx(a[:20])

    def chain():
        outs = []
        x = a
        for _ in range(6):
            x = g.gemm(x, b, cfg=cfg)
            outs += [x, g.gemm_mx(small, w), g.gemm_mx(g.quantize_mx(x), w)]
        return outs

    want = []
    x = a
    for _ in range(6):
        x = g.gemm(x, b, cfg=cfg)
        torch.cuda.synchronize()
        q = g.quantize_mx(x)
        torch.cuda.synchronize()
        want += [x, g.gemm_mx(small, w), g.gemm_mx(q, w)]
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w_) for o, w_ in zip(got, want))
    assert g.device_status()[0] == api.STATUS_OK


@pytest.mark.gpu
def test_two_streams_at_once():
    """Passes on two streams without any wait between them: nothing is shared."""
    gen = torch.Generator().manual_seed(6)
    xs = [torch.randn(m, 2048, generator=gen).bfloat16().cuda() for m in (8, 100, 300, 700)]
    ws = [g.quantize_mx((torch.randn(n, 2048, generator=gen) * 0.02).bfloat16().cuda(), "mxfp4") for n in (640, 1000)]
    want = [[g.gemm_mx(g.quantize_mx(x), w) for x in xs] for w in ws]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ws]
    got = [[], []]
    for _ in range(4):
        for x in xs:
            for i, (s, w) in enumerate(zip(streams, ws)):
                got[i].append(g.gemm_mx(g.quantize_mx(x, stream=s), w, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        for j, out in enumerate(got[i]):
            assert torch.equal(out, want[i][j % len(xs)])
    assert g.device_status()[0] == api.STATUS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_beyond_32_bits(fmt):
    """A matrix of more than 2^32 elements: its first and last rows both ways, read back, and multiplied."""
    R, C = 131077, 32808
    x = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for r in range(0, R, 16384):
        x[r:r + 16384] = torch.randn(min(16384, R - r), C, generator=gen, device="cuda")
    q, qt = g.quantize_mx_both(x, fmt)
    rows = [0, 1, 65535, 65536, R - 130, R - 1]
    value = quantise_ref(to64(x[rows]), fmt)[2]
    back = g.dequantize_mx(q)
    np.testing.assert_array_equal(to64(back[rows]), value)
    cols = [0, 5, 16384, C - 1]
    value_t = quantise_ref(to64(x[:, cols]).T.copy(), fmt)[2]
    back = g.dequantize_mx(qt)
    np.testing.assert_array_equal(to64(back[cols]), value_t)
    del back, x
    a = g.quantize_mx(torch.randn(3, C, generator=gen, device="cuda").bfloat16(), fmt)
    av = to64(g.dequantize_mx(a))
    out = g.gemm_mx(a, q)
    ref = av @ value.T
    assert (np.abs(to64(out[:, rows]) - ref) <= product_bound(av, value, ref, torch.bfloat16)).all()
    out = g.gemm_mx(q, a)  # the long side as rows of C
    assert (np.abs(to64(out[rows]) - ref.T) <= product_bound(value, av, ref.T, torch.bfloat16)).all()

"""Microscaled 4-bit floating point: quantisation, its inverse and the product, over the C ABI.

Two formats of e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives): ``"mxfp4"`` has one power-of-two
scale per 32 elements of a row, ``"nvfp4"`` one e4m3 scale per 16 and a power of two for the whole
matrix. include/b200_gemm.h defines the memory layout and the rounding.

The products of a linear layer y = x w^T and of its gradients contract over three different axes, and
blocks have to run along the contraction::

    xr, xc = quantize_mx_both(x)            # [M, K] and its transpose's form [K, M]
    wr, wc = quantize_mx_both(w)            # [N, K], [K, N]
    y  = gemm_mx(xr, wr)                    # [M, N], over K
    dr, dc = quantize_mx_both(dy)           # [M, N], [N, M]
    dx = gemm_mx(dr, wc)                    # [M, K], over N
    dw = gemm_mx(dc, xc)                    # [N, K], over M
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass

from . import api
from .api import STATUS_INVALID_ARG, GemmError

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_GROUPS = {"mxfp4": 2, "nvfp4": 4}  # 512-byte scale groups of a 128 x 256 tile


def _invalid(message: str) -> GemmError:
    return GemmError(STATUS_INVALID_ARG, message)


def _format(name) -> int:
    if name not in FORMATS:
        raise _invalid(f"format must be one of {sorted(FORMATS)}, got {name!r}")
    return FORMATS[name]


@dataclass
class MxTensor:
    """A [rows, cols] matrix in microscaled 4-bit form: ``data`` [rows, pitch] and ``scales`` [bytes],
    both uint8 CUDA tensors in the layout of include/b200_gemm.h. ``tensor_scale`` is the power of two
    (any positive number for matrices that come from elsewhere) all values are multiplied with."""
    data: object
    scales: object
    rows: int
    cols: int
    format: str = "mxfp4"
    tensor_scale: float = 1.0

    def __post_init__(self):
        import torch
        fmt = _format(self.format)
        lib = api.library()
        if self.rows <= 0 or self.cols <= 0:
            raise _invalid("rows and cols must be positive")
        for name, t, need in (("data", self.data, lib.b200_mx_data_bytes(self.rows, self.cols)),
                              ("scales", self.scales, lib.b200_mx_scale_bytes(fmt, self.rows, self.cols))):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or not t.is_contiguous():
                raise _invalid(f"{name} must be a contiguous uint8 tensor")
            if t.numel() != need:
                raise _invalid(f"{name} must hold {need} bytes for [{self.rows}, {self.cols}] {self.format}, "
                               f"got {t.numel()}")
            if t.data_ptr() % 16:
                raise _invalid(f"{name} must start on 16 bytes")
        if self.data.device != self.scales.device:
            raise _invalid("data and scales must be on one device")
        if not (self.tensor_scale > 0 and math.isfinite(self.tensor_scale)):
            raise _invalid("tensor_scale must be positive and finite")
        if self.format == "mxfp4" and self.tensor_scale != 1.0:
            raise _invalid("mxfp4 has no tensor scale (it must be 1)")

    @property
    def device(self):
        return self.data.device

    @classmethod
    def from_parts(cls, codes, block_scales, cols: int, format: str = "mxfp4", tensor_scale: float = 1.0) -> "MxTensor":
        """Lays out weights that come as packed codes [rows, ceil(cols / 2)] and plain block scales
        [rows, ceil(cols / block)] (uint8 or the 8-bit float's own type), once."""
        import torch
        _format(format)
        rows = codes.shape[0]
        blocks = -(-cols // BLOCK[format])
        if codes.dim() != 2 or block_scales.dim() != 2 or codes.shape[1] != (cols + 1) // 2 or \
                tuple(block_scales.shape) != (rows, blocks):
            raise _invalid(f"codes must be [rows, {(cols + 1) // 2}] and block_scales [rows, {blocks}]")
        if codes.element_size() != 1 or block_scales.element_size() != 1:
            raise _invalid("codes and block_scales must be 8-bit tensors")
        codes, block_scales = codes.view(torch.uint8), block_scales.view(torch.uint8)
        pitch = ((cols + 1) // 2 + 15) // 16 * 16
        data = torch.zeros(rows, pitch, dtype=torch.uint8, device=codes.device)
        data[:, :codes.shape[1]] = codes
        if cols % 2:
            data[:, cols // 2] &= 15
        row_tiles, col_tiles, groups = -(-rows // 128), -(-cols // 256), _GROUPS[format]
        s = torch.zeros(row_tiles * 128, col_tiles * groups * 4, dtype=torch.uint8, device=codes.device)
        s[:rows, :blocks] = block_scales
        s = s.view(row_tiles, 4, 32, col_tiles, groups, 4).permute(0, 3, 4, 2, 1, 5).reshape(-1)
        return cls(data, s.contiguous(), rows, cols, format, tensor_scale)

    def to_parts(self):
        """The inverse of ``from_parts``: (codes [rows, ceil(cols / 2)], block_scales [rows, blocks]), uint8."""
        row_tiles, col_tiles, groups = -(-self.rows // 128), -(-self.cols // 256), _GROUPS[self.format]
        s = self.scales.view(row_tiles, col_tiles, groups, 32, 4, 4).permute(0, 4, 3, 1, 2, 5)
        s = s.reshape(row_tiles * 128, -1)[:self.rows, :-(-self.cols // BLOCK[self.format])]
        return self.data.view(self.rows, -1)[:, :(self.cols + 1) // 2].contiguous(), s.contiguous()


@contextlib.contextmanager
def _on(device, stream):
    """Runs a call on the tensors' device and, for memory it allocates, in the order of its stream; gives
    the stream as the C ABI takes it."""
    import torch
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream().cuda_stream or None
            return
        handle = getattr(stream, "cuda_stream", stream) or 0
        if handle == torch.cuda.default_stream().cuda_stream:
            outer = torch.cuda.default_stream()
        else:
            outer = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(handle)
        if outer.device != torch.device(device):
            raise _invalid(f"the stream belongs to {outer.device}, the tensors to {device}")
        with torch.cuda.stream(outer):
            yield handle or None


def _require_cuda(t, name: str, device=None):
    if not t.is_cuda:
        raise _invalid(f"{name} must be a CUDA tensor (no CPU fallback exists)")
    if device is not None and t.device != device:
        raise _invalid(f"{name} is on {t.device}, expected {device}")


def _half_type(dtype, name: str) -> int:
    import torch
    if dtype not in (torch.bfloat16, torch.float16):
        raise _invalid(f"{name} must be bfloat16 or float16, got {dtype}")
    return int(dtype == torch.float16)


def _quantize(x, format, tensor_scale, out, out_t, rows: bool, cols: bool, stream):
    import torch
    fmt = _format(format)
    f16 = _half_type(x.dtype, "x")
    if x.dim() != 2 or x.shape[0] == 0 or x.shape[1] == 0:
        raise _invalid("x must be a 2-D tensor with at least one row and one column")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise _invalid("the columns of x must be contiguous (its rows may be any distance apart)")
    R, C = x.shape
    ld = x.stride(0) if R > 1 else C
    if ld < C:
        raise _invalid("the rows of x overlap")
    _require_cuda(x, "x")
    with _on(x.device, stream) as s:
        lib = api.library()

        def target(given, r, c, name):
            if given is None:
                data = torch.empty((r, lib.b200_mx_data_bytes(1, c)), dtype=torch.uint8, device=x.device)
                scales = torch.empty(lib.b200_mx_scale_bytes(fmt, r, c), dtype=torch.uint8, device=x.device)
                return MxTensor(data, scales, r, c, format, tensor_scale)
            if (given.rows, given.cols, given.format) != (r, c, format) or given.tensor_scale != tensor_scale:
                raise _invalid(f"{name} must be a [{r}, {c}] {format} matrix with tensor scale {tensor_scale}")
            _require_cuda(given.data, name, x.device)
            return given

        q = target(out, R, C, "out") if rows else None
        qt = target(out_t, C, R, "out") if cols else None
        ptr = lambda m: (m.data.data_ptr(), m.scales.data_ptr()) if m is not None else (None, None)  # noqa: E731
        api._check(lib.b200_mx_quantize(fmt, f16, R, C, x.data_ptr(), ld, tensor_scale, *ptr(q), *ptr(qt), s))
    return q, qt


def quantize_mx(x, format: str = "mxfp4", transpose: bool = False, tensor_scale: float = 1.0, out=None,
                stream=None) -> MxTensor:
    """The 4-bit form of x [R, C] (bf16 or fp16; rows may be strided), blocks along its rows; with
    ``transpose`` the 4-bit form of its transpose [C, R]. ``tensor_scale`` (nvfp4): a power of two near
    the matrix' largest magnitude / 2688, or 1 for values of ordinary size; block scales below 2^-9 of
    it are lost. ``out`` takes an MxTensor of the same shape and format to write into."""
    q, qt = _quantize(x, format, tensor_scale, out, out, not transpose, transpose, stream)
    return qt if transpose else q


def quantize_mx_both(x, format: str = "mxfp4", tensor_scale: float = 1.0, stream=None):
    """``(quantize_mx(x), quantize_mx(x, transpose=True))`` in one pass over x."""
    return _quantize(x, format, tensor_scale, None, None, True, True, stream)


def dequantize_mx(q: MxTensor, dtype=None, out=None, stream=None):
    """The values of q as a [rows, cols] bf16 (default) or fp16 tensor."""
    import torch
    dtype = dtype or (out.dtype if out is not None else torch.bfloat16)
    f16 = _half_type(dtype, "dtype")
    _require_cuda(q.data, "q")
    with _on(q.device, stream) as s:
        if out is None:
            out = torch.empty((q.rows, q.cols), dtype=dtype, device=q.device)
        _require_cuda(out, "out", q.device)
        if out.dtype != dtype or tuple(out.shape) != (q.rows, q.cols) or (q.cols > 1 and out.stride(1) != 1):
            raise _invalid(f"out must be a [{q.rows}, {q.cols}] {dtype} tensor with contiguous columns")
        ld = out.stride(0) if q.rows > 1 else q.cols
        if ld < q.cols:
            raise _invalid("the rows of out overlap")
        api._check(api.library().b200_mx_dequantize(_format(q.format), f16, q.rows, q.cols, q.data.data_ptr(),
                                                    q.scales.data_ptr(), q.tensor_scale, out.data_ptr(), ld, s))
    return out


def gemm_mx(a: MxTensor, b: MxTensor, out=None, alpha: float = 1.0, beta: float = 0.0, dtype=None, stream=None):
    """out[M, N] = (a[M, K] @ b[N, K]^T) * alpha + beta for two 4-bit matrices of one format, tensor scales
    applied; bf16 (default) or fp16 output, fp32 accumulation."""
    import torch
    dtype = dtype or (out.dtype if out is not None else torch.bfloat16)
    f16 = _half_type(dtype, "dtype")
    if a.format != b.format:
        raise _invalid(f"a is {a.format}, b is {b.format}")
    if a.cols != b.cols:
        raise _invalid("a and b disagree on K")
    _require_cuda(a.data, "a")
    _require_cuda(b.data, "b", a.device)
    scale = float(alpha) * a.tensor_scale * b.tensor_scale
    with _on(a.device, stream) as s:
        if out is None:
            out = torch.empty((a.rows, b.rows), dtype=dtype, device=a.device)
        _require_cuda(out, "out", a.device)
        if out.dtype != dtype or tuple(out.shape) != (a.rows, b.rows) or not out.is_contiguous():
            raise _invalid(f"out must be a contiguous [{a.rows}, {b.rows}] {dtype} tensor")
        api._check(api.library().b200_gemm_mx(_format(a.format), f16, a.rows, b.rows, a.cols, a.data.data_ptr(),
                                              a.scales.data_ptr(), b.data.data_ptr(), b.scales.data_ptr(),
                                              out.data_ptr(), scale, beta, s))
    return out

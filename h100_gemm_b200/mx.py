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

No call here records a history: results of tensors that require gradients do not, and a backward pass is made of the
calls above (in a torch.autograd.Function of the caller's, for instance).
"""
from __future__ import annotations

import contextlib
import ctypes
import math

from . import api
from .api import STATUS_INVALID_ARG, GemmError


class _Torch:
    """Stands for torch in a module until something of it is needed there: importing the package must not import it,
    and an import statement in every call costs a quarter of a microsecond."""

    def __init__(self, module: dict):
        self._module = module

    def __getattr__(self, name):
        import torch
        self._module["torch"] = torch
        return getattr(torch, name)


torch = _Torch(globals())

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAX_SIZE = 2 ** 31 - 1  # rows and columns are 32-bit numbers in the C ABI
FP32_MIN, FP32_MAX = 2.0 ** -126, 2.0 ** 128 - 2.0 ** 104  # its normal numbers
_GROUPS = {"mxfp4": 2, "nvfp4": 4}  # 512-byte scale groups of a 128 x 256 tile


def _invalid(message: str) -> GemmError:
    return GemmError(STATUS_INVALID_ARG, message)


def _format(name) -> int:
    fmt = FORMATS.get(name)
    if fmt is None:
        raise _invalid(f"format must be one of {sorted(FORMATS)}, got {name!r}")
    return fmt


def _pitch(cols: int) -> int:
    """b200_mx_data_bytes of one row."""
    return ((cols + 1) // 2 + 15) // 16 * 16


def _scale_bytes(format: str, rows: int, cols: int) -> int:
    """b200_mx_scale_bytes."""
    return ((rows + 127) // 128) * ((cols + 255) // 256) * (_GROUPS[format] * 512)


class MxTensor:
    """A [rows, cols] matrix in microscaled 4-bit form: ``data`` [rows, pitch] and ``scales`` [bytes],
    both uint8 CUDA tensors in the layout of include/b200_gemm.h. ``tensor_scale`` is the power of two
    (any positive number for matrices that come from elsewhere) all values are multiplied with."""

    __slots__ = ("rows", "cols", "format", "tensor_scale", "device", "_data", "_scales", "_pool", "_data_ptr", "_scales_ptr")

    def __init__(self, data, scales, rows: int, cols: int, format: str = "mxfp4", tensor_scale: float = 1.0):
        _format(format)
        if rows <= 0 or cols <= 0:
            raise _invalid("rows and cols must be positive")
        if rows > MAX_SIZE or cols > MAX_SIZE:
            raise _invalid(f"at most {MAX_SIZE} rows and columns, got [{rows}, {cols}]")
        if not FP32_MIN <= tensor_scale < 3.4e38:
            raise _invalid("tensor_scale must be a positive normal number in fp32")
        if format == "mxfp4" and tensor_scale != 1.0:
            raise _invalid("mxfp4 has no tensor scale (it must be 1)")
        pointers = []
        for name, t, need in (("data", data, rows * _pitch(cols)), ("scales", scales, _scale_bytes(format, rows, cols))):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.uint8 or not t.is_contiguous():
                raise _invalid(f"{name} must be a contiguous uint8 tensor")
            if t.numel() != need:
                raise _invalid(f"{name} must hold {need} bytes for [{rows}, {cols}] {format}, got {t.numel()}")
            pointers.append(t.data_ptr())
            if pointers[-1] % 16:
                raise _invalid(f"{name} must start on 16 bytes")
        if data.device != scales.device:
            raise _invalid("data and scales must be on one device")
        self.rows, self.cols, self.format, self.tensor_scale, self.device = rows, cols, format, tensor_scale, data.device
        self._data, self._scales, self._pool = data, scales, None
        self._data_ptr, self._scales_ptr = pointers

    @classmethod
    def _empty(cls, rows: int, cols: int, format: str, tensor_scale: float, device) -> "MxTensor":
        """Uninitialised, in one allocation; the two tensors are made when somebody asks for them."""
        self = cls.__new__(cls)
        codes = rows * _pitch(cols)
        at = (codes + 255) // 256 * 256
        self._pool = torch.empty(at + _scale_bytes(format, rows, cols), dtype=torch.uint8, device=device)
        self.rows, self.cols, self.format, self.tensor_scale, self.device = rows, cols, format, tensor_scale, device
        self._data = self._scales = None
        self._data_ptr = self._pool.data_ptr()
        self._scales_ptr = self._data_ptr + at
        return self

    def __reduce__(self):
        """Copies and pickles hold the tensors; the addresses that kernels get are theirs, not this object's."""
        return type(self), (self.data, self.scales, self.rows, self.cols, self.format, self.tensor_scale)

    @property
    def data(self):
        if self._data is None:
            self._data = self._pool[:self.rows * _pitch(self.cols)].view(self.rows, -1)
        return self._data

    @property
    def scales(self):
        if self._scales is None:
            self._scales = self._pool[self._scales_ptr - self._data_ptr:]
        return self._scales

    def __repr__(self):
        return f"MxTensor([{self.rows}, {self.cols}], {self.format}, tensor_scale={self.tensor_scale}, device={self.device})"

    @classmethod
    def from_parts(cls, codes, block_scales, cols: int, format: str = "mxfp4", tensor_scale: float = 1.0) -> "MxTensor":
        """Lays out weights that come as packed codes [rows, ceil(cols / 2)] and plain block scales
        [rows, ceil(cols / block)] (uint8 or the 8-bit float's own type), once."""
        _format(format)
        blocks = -(-cols // BLOCK[format])
        if codes.dim() != 2 or block_scales.dim() != 2 or codes.shape[1] != (cols + 1) // 2 or \
                tuple(block_scales.shape) != (codes.shape[0], blocks):
            raise _invalid(f"codes must be [rows, {(cols + 1) // 2}] and block_scales [rows, {blocks}]")
        if codes.element_size() != 1 or block_scales.element_size() != 1:
            raise _invalid("codes and block_scales must be 8-bit tensors")
        rows = codes.shape[0]
        codes, block_scales = codes.view(torch.uint8), block_scales.view(torch.uint8)
        data = torch.zeros(rows, _pitch(cols), dtype=torch.uint8, device=codes.device)
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
def _elsewhere(device, stream):
    """Another device than the current one, or a stream of the caller's choice: memory is allocated there, in
    that stream's order."""
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream().cuda_stream or None
            return
        handle = getattr(stream, "cuda_stream", stream) or 0
        if handle == torch.cuda.default_stream().cuda_stream:
            outer = torch.cuda.default_stream()
        else:
            outer = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(handle)
        if getattr(stream, "device", outer.device) != device:
            raise _invalid(f"the stream belongs to {stream.device}, the tensors to {device}")
        with torch.cuda.stream(outer):
            yield handle or None


def _current(device, stream):
    """The current stream's handle where a call can run as it is, the usual case; else False (see _elsewhere)."""
    if stream is None:
        index = device.index
        if torch._C._cuda_getDevice() == index:
            return torch._C._cuda_getCurrentRawStream(index) or None
    return False


def _require_cuda(device, name: str, expected=None):
    if device.type != "cuda":
        raise _invalid(f"{name} must be a CUDA tensor (no CPU fallback exists)")
    if expected is not None and device != expected:
        raise _invalid(f"{name} is on {device}, expected {expected}")


def _half_type(dtype, name: str) -> int:
    if dtype is torch.bfloat16:
        return 0
    if dtype is torch.float16:
        return 1
    raise _invalid(f"{name} must be bfloat16 or float16, got {dtype}")


def _row_stride(t, name: str) -> int:
    """Elements between the rows of a 2-D tensor whose columns are contiguous."""
    rows, cols = t.shape
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise _invalid(f"the columns of {name} must be contiguous (its rows may be any distance apart)")
    if rows == 1:
        return cols
    if ld < cols:
        raise _invalid(f"the rows of {name} overlap")
    return ld


def _quantize(x, format, tensor_scale, out, rows: bool, cols: bool, stream):
    fmt = _format(format)
    f16 = _half_type(x.dtype, "x")
    if x.dim() != 2 or x.numel() == 0:
        raise _invalid("x must be a 2-D tensor with at least one row and one column")
    if max(x.shape) > MAX_SIZE:
        raise _invalid(f"at most {MAX_SIZE} rows and columns, got {list(x.shape)}")
    ld = _row_stride(x, "x")
    device = x.device
    _require_cuda(device, "x")
    if format == "mxfp4" and tensor_scale != 1.0:
        raise _invalid("mxfp4 has no tensor scale (it must be 1)")
    if out is not None:
        want = tuple(x.shape) if rows else tuple(x.shape)[::-1]
        if (out.rows, out.cols) != want or out.format != format or out.tensor_scale != tensor_scale:
            raise _invalid(f"out must be a [{want[0]}, {want[1]}] {format} matrix with tensor scale {tensor_scale}")
        _require_cuda(out.device, "out", device)
    handle = _current(device, stream)
    if handle is not False:
        return _launch_quantize(x, fmt, f16, ld, format, tensor_scale, out, rows, cols, handle)
    with _elsewhere(device, stream) as handle:
        return _launch_quantize(x, fmt, f16, ld, format, tensor_scale, out, rows, cols, handle)


def _launch_quantize(x, fmt, f16, ld, format, tensor_scale, out, rows, cols, handle):
    R, C = x.shape
    q = qt = data = scales = data_t = scales_t = None
    if rows:
        q = out or MxTensor._empty(R, C, format, tensor_scale, x.device)
        data, scales = q._data_ptr, q._scales_ptr
    if cols:
        qt = out or MxTensor._empty(C, R, format, tensor_scale, x.device)
        data_t, scales_t = qt._data_ptr, qt._scales_ptr
    rc = api.library().b200_mx_quantize(fmt, f16, R, C, x.data_ptr(), ld, tensor_scale, data, scales, data_t, scales_t, handle)
    if rc:
        api._check(rc)
    return q, qt


def quantize_mx(x, format: str = "mxfp4", transpose: bool = False, tensor_scale: float = 1.0, out=None,
                stream=None) -> MxTensor:
    """The 4-bit form of x [R, C] (bf16 or fp16; rows may be strided), blocks along its rows; with
    ``transpose`` the 4-bit form of its transpose [C, R]. ``tensor_scale`` (nvfp4): a power of two near
    the matrix' largest magnitude / 2688, or 1 for values of ordinary size; block scales below 2^-9 of
    it are lost. ``out`` takes an MxTensor of the same shape and format to write into."""
    q, qt = _quantize(x, format, tensor_scale, out, not transpose, transpose, stream)
    return qt if transpose else q


def quantize_mx_both(x, format: str = "mxfp4", tensor_scale: float = 1.0, stream=None):
    """``(quantize_mx(x), quantize_mx(x, transpose=True))`` in one pass over x."""
    return _quantize(x, format, tensor_scale, None, True, True, stream)


def _output(out, shape, dtype, device, contiguous: bool) -> None:
    _require_cuda(out.device, "out", device)
    if out.dtype is not dtype or out.shape != shape or (contiguous and not out.is_contiguous()):
        raise _invalid(f"out must be a {'contiguous ' if contiguous else ''}{list(shape)} {dtype} tensor")


def dequantize_mx(q: MxTensor, dtype=None, out=None, stream=None):
    """The values of q as a [rows, cols] bf16 (default) or fp16 tensor."""
    if not isinstance(q, MxTensor):
        raise _invalid(f"q must be an MxTensor, got {type(q).__name__}")
    dtype = dtype or (out.dtype if out is not None else torch.bfloat16)
    f16 = _half_type(dtype, "dtype")
    device = q.device
    _require_cuda(device, "q")
    if out is not None:
        _output(out, (q.rows, q.cols), dtype, device, False)

    ld = q.cols if out is None else _row_stride(out, "out")
    handle = _current(device, stream)
    if handle is not False:
        return _launch_dequantize(q, dtype, f16, out, ld, handle)
    with _elsewhere(device, stream) as handle:
        return _launch_dequantize(q, dtype, f16, out, ld, handle)


def _launch_dequantize(q, dtype, f16, out, ld, handle):
    if out is None:
        out = torch.empty(q.rows, q.cols, dtype=dtype, device=q.device)
    rc = api.library().b200_mx_dequantize(FORMATS[q.format], f16, q.rows, q.cols, q._data_ptr, q._scales_ptr, q.tensor_scale,
                                          out.data_ptr(), ld, handle)
    if rc:
        api._check(rc)
    return out


def _unusual_factor(factor: float, alpha: float) -> None:
    """Raises where alpha times the tensor scales is not what fp32 can hold. (An alpha of zero, an infinite or a NaN one
    mean what they say, and a small power of two is exact.)"""
    if alpha == 0 or not math.isfinite(alpha) or (abs(factor) < 1 and ctypes.c_float(factor).value == factor):
        return
    raise _invalid(f"alpha times the tensor scales of a and b is {factor}, outside fp32's range: leave a power of two of it to the caller")


def gemm_mx(a: MxTensor, b: MxTensor, out=None, alpha: float = 1.0, beta: float = 0.0, dtype=None, stream=None):
    """out[M, N] = (a[M, K] @ b[N, K]^T) * alpha + beta for two 4-bit matrices of one format, tensor scales
    applied (their product with alpha has to be within fp32's range); bf16 (default) or fp16 output, fp32
    accumulation."""
    if not isinstance(a, MxTensor) or not isinstance(b, MxTensor):
        raise _invalid(f"a and b must be MxTensors, got {type(a).__name__} and {type(b).__name__}")
    dtype = dtype or (out.dtype if out is not None else torch.bfloat16)
    f16 = _half_type(dtype, "dtype")
    if a.format != b.format:
        raise _invalid(f"a is {a.format}, b is {b.format}")
    if a.cols != b.cols:
        raise _invalid("a and b disagree on K")
    factor = alpha * a.tensor_scale * b.tensor_scale
    if not FP32_MIN <= abs(factor) <= FP32_MAX:
        _unusual_factor(factor, alpha)
    device = a.device
    _require_cuda(device, "a")
    _require_cuda(b.device, "b", device)
    if out is not None:
        _output(out, (a.rows, b.rows), dtype, device, True)

    handle = _current(device, stream)
    if handle is not False:
        return _launch_gemm(a, b, dtype, f16, out, factor, beta, handle)
    with _elsewhere(device, stream) as handle:
        return _launch_gemm(a, b, dtype, f16, out, factor, beta, handle)


def _launch_gemm(a, b, dtype, f16, out, factor, beta, handle):
    if out is None:
        out = torch.empty(a.rows, b.rows, dtype=dtype, device=a.device)
    rc = api.library().b200_gemm_mx(FORMATS[a.format], f16, a.rows, b.rows, a.cols, a._data_ptr, a._scales_ptr, b._data_ptr,
                                    b._scales_ptr, out.data_ptr(), factor, beta, handle)
    if rc:
        api._check(rc)
    return out

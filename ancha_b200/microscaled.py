"""Linear layers in 8 and 4 bits: microscaled arrays over torch CUDA tensors.

A :class:`Microscaled` array holds rows of 8-bit or 4-bit floating-point elements with one scale for
each block of a row. ``FORMATS`` names the number formats:

* ``"mxf8"``: E4M3 elements, a power of two for each 32;
* ``"mxf4"``: E2M1 elements, a power of two for each 32;
* ``"nvf4"``: E2M1 elements, an E4M3 scale for each 16 and one f32 scale of the whole array.

:func:`quantize` and :func:`dequantize` go to them and back, :func:`add_rms_norm` adds to the residual
stream and writes its RMS norm quantised, and :func:`linear` multiplies two arrays on the block-scaled
tensor cores (``fused.linear`` is the 16-bit and 32-bit form). A pre-norm feed-forward block is ::

    q, stream = add_rms_norm(branch, stream, gain, format="mxf8")
    hidden = linear(q, w1, b1, "gelu", format="mxf8")
    branch = linear(hidden, w2, b2, dtype=torch.bfloat16)

The functions run on the stream that is torch's current one on the tensors' device, allocate only what
they return, keep nothing between calls and never synchronise, so they can be captured into CUDA graphs.
They raise ``AnchaError`` for arguments they do not take; ``fused.check_device`` raises it where a kernel has
given up a device-side wait. No gradients: this is an inference engine.
"""
from __future__ import annotations

import functools
from ctypes import byref
from typing import Optional

import torch

from . import _native as N

FORMATS = {"mxf8": N.MXF8, "mxf4": N.MXF4, "nvf4": N.NVF4}
BLOCK = {"mxf8": 32, "mxf4": 32, "nvf4": 16}
ACTIVATIONS = {"none": N.ACT_NONE, "gelu": N.ACT_GELU, "tanh": N.ACT_TANH}
_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


def _invalid(message: str) -> N.AnchaError:
    return N.AnchaError(N.E_INVALID, message)


@functools.lru_cache(maxsize=256)
def _layout(fmt: str, rows: int, cols: int):
    """(bytes from row to row, shape of the scales, bytes of the elements, bytes of the scales):
    ``ancha_mx_layout``'s rule."""
    if fmt not in FORMATS:
        raise _invalid(f"unknown format {fmt!r}: one of {', '.join(FORMATS)}")
    if cols < 1 or rows < 0:
        raise _invalid("rows without elements, or a negative number of rows")
    ld = -(-(cols if fmt == "mxf8" else (cols + 1) // 2) // 16) * 16
    mt, kt = -(-rows // 128), -(-cols // (4 * BLOCK[fmt]))
    return ld, (mt, kt, 32, 4, 4), rows * ld, mt * kt * 512


class Microscaled:
    """Rows of quantised elements.

    ``data``: uint8 ``[rows, ld]``, elements in memory order (two per byte in the 4-bit formats, the even
    column in the low half), ``ld`` a multiple of 16. ``scales``: uint8 ``[rows / 128, blocks / 4, 32, 4, 4]``
    (both rounded up): the code of (row, block) at ``[row // 128, block // 4, row % 32, row % 128 // 32,
    block % 4]``. ``global_scale``: one f32 on the device (``nvf4`` only; None is 1).
    """
    __slots__ = ("format", "rows", "cols", "global_scale", "_data", "_scales", "_buffer")

    def __init__(self, format: str, rows: int, cols: int, data: torch.Tensor, scales: torch.Tensor,
                 global_scale: Optional[torch.Tensor] = None):
        self.format, self.rows, self.cols, self.global_scale = format, rows, cols, global_scale
        self._data, self._scales, self._buffer = data, scales, None

    @classmethod
    def _new(cls, format, rows, cols, like, global_scale):
        """An array in one new allocation on the device of ``like``: elements, then scales."""
        q = object.__new__(cls)
        q.format, q.rows, q.cols, q.global_scale = format, rows, cols, global_scale
        _, _, data, scales = _layout(format, rows, cols)
        q._buffer = like.new_empty(data + scales, dtype=torch.uint8)
        q._data = q._scales = None
        return q

    @property
    def data(self) -> torch.Tensor:
        if self._data is None:
            ld = _layout(self.format, self.rows, self.cols)[0]
            self._data = self._buffer.as_strided((self.rows, ld), (ld, 1), 0)
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            _, shape, offset, _ = _layout(self.format, self.rows, self.cols)
            self._scales = self._buffer.as_strided(shape, (shape[1] * 512, 512, 16, 4, 1), offset)
        return self._scales

    def scale_codes(self) -> torch.Tensor:
        """The scale codes as a uint8 ``[rows, blocks]`` matrix (a copy)."""
        s = self.scales
        blocks = -(-self.cols // BLOCK[self.format])
        return s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, -1)[:self.rows, :blocks]


def empty(format: str, rows: int, cols: int, device="cuda", global_scale=None) -> Microscaled:
    """An array with memory for ``rows`` by ``cols`` elements, not yet written."""
    return Microscaled._new(format, rows, cols, torch.empty(0, device=device), global_scale)


def _device(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise _invalid("tensors must be on a CUDA device")
    return t.get_device()


def _on(t, device: int, name: str):
    if t.get_device() != device:
        raise _invalid(f"{name}: not on the device of the first operand")


def _vector(t, device: int, n: int, name: str):
    """Address of a contiguous f32 vector of n elements, None for None."""
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise _invalid(f"{name}: needs {n} contiguous f32 elements")
    _on(t, device, name)
    return t.data_ptr()


def _matrix(t, device: int, name: str):
    """(dtype code, row stride) of a 2-D tensor whose rows are dense."""
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise _invalid(f"{name}: unsupported dtype {t.dtype}")
    if t.dim() != 2:
        raise _invalid(f"{name}: needs two axes")
    if t.get_device() != device:
        raise _invalid(f"{name}: not on the device of the first operand")
    if t.is_contiguous():  # the stride of a single row is arbitrary in torch
        return code, t.shape[1] or 1
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise _invalid(f"{name}: its last axis must be contiguous")
    return code, (t.stride(0) if rows > 1 else cols)


def _array(q: Microscaled, device: int, name: str) -> N.MxArray:
    fmt, rows, cols = q.format, q.rows, q.cols
    ld, shape, data_bytes, _ = _layout(fmt, rows, cols)
    g = q.global_scale
    if g is not None:
        g = _vector(g, device, 1, f"{name}: global_scale")
    buffer = q._buffer
    if buffer is not None:
        if buffer.get_device() != device:
            raise _invalid(f"{name}: not on the device of the first operand")
        at = buffer.data_ptr()
        return N.MxArray(FORMATS[fmt], rows, cols, at, ld, at + data_bytes, g)
    data, scales = q._data, q._scales
    if data.dtype is not torch.uint8 or data.shape != (rows, ld) or not data.is_contiguous():
        if data.dtype is not torch.uint8 or data.dim() != 2 or data.shape[0] != rows or data.shape[1] < ld \
                or data.stride(1) != 1:
            raise _invalid(f"{name}: data is not uint8 [{rows}, >= {ld}] with contiguous rows")
        if rows > 1:
            ld = data.stride(0)
    if scales.dtype is not torch.uint8 or scales.shape != shape or not scales.is_contiguous():
        raise _invalid(f"{name}: scales are not contiguous uint8 {shape}")
    if data.get_device() != device or scales.get_device() != device:
        raise _invalid(f"{name}: not on the device of the first operand")
    return N.MxArray(FORMATS[fmt], rows, cols, data.data_ptr(), ld, scales.data_ptr(), g)


def _run(device: int, fn, *args):
    """Call the library on torch's current stream of `device`, which is made current for the call."""
    if torch._C._cuda_getDevice() == device:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        N.check(status)


def quantize(x: torch.Tensor, format: str = "mxf8", global_scale: Optional[torch.Tensor] = None) -> Microscaled:
    """Quantise the rows of ``x [rows, cols]`` (f32, bf16 or f16; any row stride). Scales and rounding as
    ``ancha_mx_quantize`` says. ``global_scale`` (``nvf4``): one f32 on the device, usually
    ``max|x| / (6 * 448)`` and at most 2^125; it becomes the array's."""
    device = _device(x)
    dtype, ld = _matrix(x, device, "x")
    rows, cols = x.shape
    out = Microscaled._new(format, rows, cols, x, global_scale)
    _run(device, N.lib().ancha_mx_quantize, x.data_ptr(), dtype, ld, byref(_array(out, device, "out")))
    return out


def dequantize(q: Microscaled, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``q`` stands for, ``[rows, cols]`` in ``dtype`` (f32, bf16 or f16)."""
    memory = q._data if q._buffer is None else q._buffer
    device = _device(memory)
    code = _DTYPES.get(dtype)
    if code is None:
        raise _invalid(f"unsupported dtype {dtype}")
    a = _array(q, device, "q")
    out = torch.empty_strided((q.rows, q.cols), (q.cols, 1), dtype=dtype, device=memory.device)
    _run(device, N.lib().ancha_mx_dequantize, byref(a), out.data_ptr(), code, q.cols)
    return out


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, gain: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, format: str = "mxf8", global_scale: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None):
    """``s = residual + x`` (``x`` without a residual), added in f32 and rounded to the residual's dtype, and the quantised rows of
    ``s / sqrt(mean(s^2) + eps) * gain``. Returns ``(Microscaled, s)``; ``s`` has the residual's dtype and
    is ``x`` itself without a residual. ``residual_out`` takes ``s`` (``residual`` itself: in place).
    ``x`` and ``residual``: f32, bf16 or f16 ``[rows, cols]``, at most 32768 columns; ``gain``: f32 ``[cols]``."""
    device = _device(x)
    dtype, ldx = _matrix(x, device, "x")
    rows, cols = x.shape
    stream, res_type, ldr, ldro, res, res_out = x, dtype, ldx, ldx, None, None
    if residual is not None:
        if residual.shape != x.shape:
            raise _invalid("residual: not the shape of x")
        res_type, ldr = _matrix(residual, device, "residual")
        res = residual.data_ptr()
        if residual_out is None:
            residual_out = torch.empty_like(residual, memory_format=torch.contiguous_format)
            stream, ldro, res_out = residual_out, cols, residual_out.data_ptr()
    if residual_out is not None and stream is x:
        if residual_out.shape != x.shape or residual_out.dtype != (x if residual is None else residual).dtype:
            raise _invalid("residual_out: not the shape and dtype of the residual stream")
        ldro = _matrix(residual_out, device, "residual_out")[1]
        stream, res_out = residual_out, residual_out.data_ptr()
    out = Microscaled._new(format, rows, cols, x, global_scale)
    _run(device, N.lib().ancha_mx_add_rms_norm_fwd, byref(N.MxNormDesc(dtype, res_type, ldx, ldr, ldro, eps)), x.data_ptr(),
         res, _vector(gain, device, cols, "gain"), res_out, byref(_array(out, device, "out")))
    return out, stream


def linear(x: Microscaled, weight: Microscaled, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
           format: Optional[str] = None, global_scale: Optional[torch.Tensor] = None):
    """``act(x [m, k] . weight [n, k]^T + bias [n]) + residual [m, n]`` of two arrays of one format, with
    f32 accumulation. ``act``: ``"none"``, ``"gelu"`` (erf) or ``"tanh"``; ``bias`` f32; ``residual`` f32, bf16
    or f16. The result is a tensor of ``dtype`` (default bf16), or with ``format`` a quantised array
    (``global_scale`` as in :func:`quantize`)."""
    memory = x._data if x._buffer is None else x._buffer
    device = _device(memory)
    if act not in ACTIVATIONS:
        raise _invalid(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
    m, n = x.rows, weight.rows
    res, res_type, ldr = None, N.F32, 0
    if residual is not None:
        if residual.shape != (m, n):
            raise _invalid("residual: not the shape of the product")
        res_type, ldr = _matrix(residual, device, "residual")
        res = residual.data_ptr()
    a, w, b = _array(x, device, "x"), _array(weight, device, "weight"), _vector(bias, device, n, "bias")
    if format is not None:
        if dtype is not None:
            raise _invalid("dtype and format exclude each other")
        out = Microscaled._new(format, m, n, memory, global_scale)
        _run(device, N.lib().ancha_mx_linear_fwd, byref(N.MxLinearDesc(ACTIVATIONS[act], N.F32, res_type, n, ldr)), byref(a),
             byref(w), b, res, None, byref(_array(out, device, "out")))
        return out
    if global_scale is not None:
        raise _invalid("global_scale without format")
    dtype = torch.bfloat16 if dtype is None else dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise _invalid(f"unsupported dtype {dtype}")
    out = torch.empty_strided((m, n), (n, 1), dtype=dtype, device=memory.device)
    _run(device, N.lib().ancha_mx_linear_fwd, byref(N.MxLinearDesc(ACTIVATIONS[act], code, res_type, n, ldr)), byref(a),
         byref(w), b, res, out.data_ptr(), None)
    return out

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
They raise ``AnchaError`` for arguments they do not take. No gradients: this is an inference engine.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as N

FORMATS = {"mxf8": N.MXF8, "mxf4": N.MXF4, "nvf4": N.NVF4}
BLOCK = {"mxf8": 32, "mxf4": 32, "nvf4": 16}
ACTIVATIONS = {"none": N.ACT_NONE, "gelu": N.ACT_GELU, "tanh": N.ACT_TANH}
_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


@dataclass(frozen=True)
class Microscaled:
    """Rows of quantised elements. ``data``: uint8 ``[rows, ld]``, elements in memory order (two per byte
    in the 4-bit formats, the even column in the low half). ``scales``: uint8 ``[rows / 128, blocks / 4,
    32, 4, 4]`` (both rounded up): the code of (row, block) at ``[row // 128, block // 4, row % 32,
    row % 128 // 32, block % 4]``. ``global_scale``: one f32 on the device (``nvf4`` only; None is 1)."""
    format: str
    rows: int
    cols: int
    data: torch.Tensor
    scales: torch.Tensor
    global_scale: Optional[torch.Tensor] = None

    def scale_codes(self) -> torch.Tensor:
        """The scale codes as a uint8 ``[rows, blocks]`` matrix (a copy)."""
        s = self.scales
        blocks = -(-self.cols // BLOCK[self.format])
        return s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, -1)[:self.rows, :blocks]


def _invalid(message: str) -> N.AnchaError:
    return N.AnchaError(N.E_INVALID, message)


def _shapes(fmt: str, rows: int, cols: int):
    """Shapes of ``data`` and ``scales`` (``ancha_mx_layout``'s rule)."""
    if fmt not in FORMATS:
        raise _invalid(f"unknown format {fmt!r}: one of {', '.join(FORMATS)}")
    if cols < 1:
        raise _invalid("rows without elements")
    ld = -(-(cols if fmt == "mxf8" else (cols + 1) // 2) // 16) * 16
    return (rows, ld), (-(-rows // 128), -(-cols // (4 * BLOCK[fmt])), 32, 4, 4)


def empty(format: str, rows: int, cols: int, device="cuda", global_scale=None) -> Microscaled:
    """An array with memory for ``rows`` by ``cols`` elements, not yet written."""
    data, scales = _shapes(format, rows, cols)
    return Microscaled(format, rows, cols, torch.empty(data, dtype=torch.uint8, device=device),
                       torch.empty(scales, dtype=torch.uint8, device=device), global_scale)


class _Call:
    """The device and stream of a call, and the check that its tensors live there."""

    def __init__(self, tensor):
        if not tensor.is_cuda:
            raise _invalid("tensors must be on a CUDA device")
        self.index = tensor.device.index

    def on(self, t, name: str):
        if not t.is_cuda or t.device.index != self.index:
            raise _invalid(f"{name}: not on the device of the first operand")
        return t

    def vector(self, t, name: str, n: int):
        """Address of a contiguous f32 vector of n elements, None for None."""
        if t is None:
            return None
        if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
            raise _invalid(f"{name}: needs {n} contiguous f32 elements")
        return self.on(t, name).data_ptr()

    def matrix(self, t, name: str):
        """(dtype code, row stride) of a 2-D tensor whose rows are dense."""
        code = _DTYPES.get(t.dtype)
        if code is None:
            raise _invalid(f"{name}: unsupported dtype {t.dtype}")
        if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
            raise _invalid(f"{name}: needs two axes, the last one contiguous")
        self.on(t, name)
        # The stride of a single row is arbitrary in torch.
        return code, (t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1))

    def array(self, q: Microscaled, name: str) -> N.MxArray:
        data, scales = _shapes(q.format, q.rows, q.cols)
        if q.data.dtype != torch.uint8 or q.data.dim() != 2 or q.data.shape[0] != q.rows \
                or q.data.shape[1] < data[1] or q.data.stride(1) != 1:
            raise _invalid(f"{name}: data is not uint8 [rows, >= {data[1]}] with contiguous rows")
        if q.scales.dtype != torch.uint8 or tuple(q.scales.shape) != scales or not q.scales.is_contiguous():
            raise _invalid(f"{name}: scales are not contiguous uint8 {scales}")
        self.on(q.data, name)
        self.on(q.scales, name)
        ld = q.data.stride(0) if q.rows > 1 else data[1]
        return N.MxArray(FORMATS[q.format], q.rows, q.cols, q.data.data_ptr(), ld, q.scales.data_ptr(),
                         self.vector(q.global_scale, f"{name}: global_scale", 1))

    def run(self, fn, *args):
        """Call the library with torch's current stream of the tensors' device, which is made current."""
        if torch.cuda.current_device() == self.index:
            N.check(fn(*args, torch.cuda.current_stream(self.index).cuda_stream))
        else:
            with torch.cuda.device(self.index):
                N.check(fn(*args, torch.cuda.current_stream(self.index).cuda_stream))


def quantize(x: torch.Tensor, format: str = "mxf8", global_scale: Optional[torch.Tensor] = None) -> Microscaled:
    """Quantise the rows of ``x [rows, cols]`` (f32, bf16 or f16; any row stride). Scales and rounding as
    ``ancha_mx_quantize`` says. ``global_scale`` (``nvf4``): one f32 on the device, usually
    ``max|x| / (6 * 448)``; it becomes the array's."""
    call = _Call(x)
    dtype, ld = call.matrix(x, "x")
    out = empty(format, x.shape[0], x.shape[1], x.device, global_scale)
    call.run(N.lib().ancha_mx_quantize, x.data_ptr(), dtype, ld, C.byref(call.array(out, "out")))
    return out


def dequantize(q: Microscaled, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``q`` stands for, ``[rows, cols]`` in ``dtype`` (f32, bf16 or f16)."""
    call = _Call(q.data)
    code = _DTYPES.get(dtype)
    if code is None:
        raise _invalid(f"unsupported dtype {dtype}")
    out = torch.empty((q.rows, q.cols), dtype=dtype, device=q.data.device)
    call.run(N.lib().ancha_mx_dequantize, C.byref(call.array(q, "q")), out.data_ptr(), code, q.cols)
    return out


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, gain: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, format: str = "mxf8", global_scale: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None):
    """``s = residual + x`` (``x`` without a residual), and the quantised rows of
    ``s / sqrt(mean(s^2) + eps) * gain``. Returns ``(Microscaled, s)``; ``s`` has the residual's dtype and
    is ``x`` itself without a residual. ``residual_out`` takes ``s`` (``residual`` itself: in place).
    ``x`` and ``residual``: f32, bf16 or f16 ``[rows, cols]``, at most 32768 columns; ``gain``: f32 ``[cols]``."""
    call = _Call(x)
    dtype, ldx = call.matrix(x, "x")
    rows, cols = x.shape
    res_type, ldr, ldro = dtype, ldx, ldx
    if residual is not None:
        if residual.shape != x.shape:
            raise _invalid("residual: not the shape of x")
        res_type, ldr = call.matrix(residual, "residual")
        if residual_out is None:
            residual_out = torch.empty((rows, cols), dtype=residual.dtype, device=x.device)
    if residual_out is not None:
        if residual_out.shape != x.shape or residual_out.dtype != (x if residual is None else residual).dtype:
            raise _invalid("residual_out: not the shape and dtype of the residual stream")
        ldro = call.matrix(residual_out, "residual_out")[1]
    out = empty(format, rows, cols, x.device, global_scale)
    desc = N.MxNormDesc(dtype, res_type, ldx, ldr, ldro, eps)
    call.run(N.lib().ancha_mx_add_rms_norm_fwd, C.byref(desc), x.data_ptr(),
             None if residual is None else residual.data_ptr(), call.vector(gain, "gain", cols),
             None if residual_out is None else residual_out.data_ptr(), C.byref(call.array(out, "out")))
    return out, (x if residual_out is None else residual_out)


def linear(x: Microscaled, weight: Microscaled, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
           format: Optional[str] = None, global_scale: Optional[torch.Tensor] = None):
    """``act(x [m, k] . weight [n, k]^T + bias [n]) + residual [m, n]`` of two arrays of one format, with
    f32 accumulation. ``act``: ``"none"``, ``"gelu"`` (erf) or ``"tanh"``; ``bias`` f32; ``residual`` f32, bf16
    or f16. The result is a tensor of ``dtype`` (default bf16), or with ``format`` a quantised array
    (``global_scale`` as in :func:`quantize`)."""
    call = _Call(x.data)
    if act not in ACTIVATIONS:
        raise _invalid(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
    if dtype is not None and format is not None:
        raise _invalid("dtype and format exclude each other")
    m, n = x.rows, weight.rows
    res_type, ldr = N.F32, 0
    if residual is not None:
        if tuple(residual.shape) != (m, n):
            raise _invalid("residual: not the shape of the product")
        res_type, ldr = call.matrix(residual, "residual")
    a, w, b = call.array(x, "x"), call.array(weight, "weight"), call.vector(bias, "bias", n)
    res = None if residual is None else residual.data_ptr()
    if format is not None:
        out = empty(format, m, n, x.data.device, global_scale)
        desc = N.MxLinearDesc(ACTIVATIONS[act], N.F32, res_type, n, ldr)
        call.run(N.lib().ancha_mx_linear_fwd, C.byref(desc), C.byref(a), C.byref(w), b, res, None,
                 C.byref(call.array(out, "out")))
        return out
    if global_scale is not None:
        raise _invalid("global_scale without format")
    dtype = torch.bfloat16 if dtype is None else dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise _invalid(f"unsupported dtype {dtype}")
    out = torch.empty((m, n), dtype=dtype, device=x.data.device)
    desc = N.MxLinearDesc(ACTIVATIONS[act], code, res_type, n, ldr)
    call.run(N.lib().ancha_mx_linear_fwd, C.byref(desc), C.byref(a), C.byref(w), b, res, out.data_ptr(), None)
    return out

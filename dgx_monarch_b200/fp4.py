"""Microscaled 4-bit floating point: packed tensors, quantisation, reading
back, and the product of two packed tensors on the tensor cores.

nvfp4 (e2m1 codes, an e4m3 scale for 16 of them, one fp32 scale for the
tensor) is the format whose activation scale the reference shares among the
ranks of a sequence-parallel call (adapters/quant_activation_scale.py:133-142;
shard.SharedActivationScale gives it); mxfp4 has a power of two for 32 codes.
There is no CPU path, and no call records an autograd graph.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._call import launch, no_graph, plan
from .ops import _dtype_code, _ptr, _require_cuda

FORMATS = {"nvfp4": _lib.FP4_NVFP4, "mxfp4": _lib.FP4_MXFP4}
BLOCK = {"nvfp4": 16, "mxfp4": 32}
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def values_shape(rows: int, cols: int) -> tuple[int, int]:
    """Two codes a byte, the even column in the low bits, rows of whole 16 bytes."""
    return rows, (cols + 31) // 32 * 16


def scales_shape(rows: int, cols: int, format: str) -> tuple[int, int, int, int, int]:
    """(row tile, block group, r % 32, r % 128 // 32, b % 4) of row r and block b."""
    return (rows + 127) // 128, -(-cols // (4 * BLOCK[format])), 32, 4, 4


def _check_format(format: str) -> int:
    if format not in FORMATS:
        raise ValueError(f"format {format!r} is not one of {sorted(FORMATS)}")
    return FORMATS[format]


class _Layout:
    """Where the parts of a packed tensor lie in one buffer, on 256 bytes each;
    the scratch of its quantisation follows them."""

    __slots__ = ("shape", "format", "rows", "cols", "scales", "scale", "scratch", "total", "devices")

    def __init__(self, shape, format: str, index: int, scratch: int) -> None:
        up = lambda n: (n + 255) // 256 * 256
        self.shape, self.format = tuple(shape), format
        self.rows, self.cols = math.prod(shape[:-1]), shape[-1]
        self.scales = up(math.prod(values_shape(self.rows, self.cols)))
        end = self.scales + up(math.prod(scales_shape(self.rows, self.cols, format)))
        self.scale = end if format == "nvfp4" else None
        self.scratch = end + (256 if format == "nvfp4" else 0)
        self.total = max(self.scratch + scratch, 256)
        self.devices = (index, index, index if format == "nvfp4" else None)


class Fp4Tensor:
    """A (..., cols) tensor in 4 bits, its leading dimensions folded into rows.

    values: uint8 of values_shape, zero past the last column; scales: uint8 of
    scales_shape, zero past a row's last block (bytes of rows past the last are not
    read; e4m3 ones have no sign, 0x7F at the most); scale: the fp32 scale of an
    nvfp4 tensor (one element on the device), None for mxfp4.  quantize_fp4 makes them; a weight kept in this layout is
    wrapped as it is."""

    __slots__ = ("shape", "format", "rows", "cols", "_values", "_scales", "_scale", "_buffer", "_offsets", "_devices")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, shape, format: str,
                 scale: torch.Tensor | None = None) -> None:
        _check_format(format)
        shape = tuple(shape)
        if not shape or shape[-1] < 1 or min(shape) < 0:
            raise ValueError(f"shape {shape} has no columns")
        rows, cols = math.prod(shape[:-1]), shape[-1]
        if values.shape != values_shape(rows, cols) or values.dtype != torch.uint8 or not values.is_contiguous():
            raise ValueError(f"values {tuple(values.shape)} {values.dtype} is not a contiguous uint8 "
                             f"{values_shape(rows, cols)} tensor")
        if (scales.shape != scales_shape(rows, cols, format) or scales.dtype != torch.uint8
                or not scales.is_contiguous()):
            raise ValueError(f"scales {tuple(scales.shape)} {scales.dtype} is not a contiguous uint8 "
                             f"{scales_shape(rows, cols, format)} tensor")
        if (scale is None) != (format == "mxfp4") or (scale is not None and (
                scale.dtype != torch.float32 or scale.numel() != 1)):
            raise ValueError("an nvfp4 tensor has one fp32 scale, an mxfp4 tensor none")
        self.shape, self.format, self.rows, self.cols = shape, format, rows, cols
        self._values, self._scales, self._scale, self._buffer, self._offsets = values, scales, scale, None, None
        self._devices = (values.get_device(), scales.get_device(), None if scale is None else scale.get_device())

    @classmethod
    def _made(cls, buffer: torch.Tensor, layout: "_Layout") -> "Fp4Tensor":
        """In one fresh buffer of layout.total bytes; its parts are views made on demand."""
        t = cls.__new__(cls)
        t.shape, t.format, t.rows, t.cols = layout.shape, layout.format, layout.rows, layout.cols
        t._values = t._scales = t._scale = None
        t._buffer, t._offsets, t._devices = buffer, layout, layout.devices
        return t

    @property
    def values(self) -> torch.Tensor:
        if self._values is None:
            shape = values_shape(self.rows, self.cols)
            self._values = self._buffer[:math.prod(shape)].view(shape)
        return self._values

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            shape, at = scales_shape(self.rows, self.cols, self.format), self._offsets.scales
            self._scales = self._buffer[at:at + math.prod(shape)].view(shape)
        return self._scales

    @property
    def scale(self) -> torch.Tensor | None:
        if self._scale is None and self._buffer is not None and self._offsets.scale is not None:
            at = self._offsets.scale
            self._scale = self._buffer[at:at + 4].view(torch.float32).view(())
        return self._scale

    @property
    def device(self) -> torch.device:
        return (self._values if self._buffer is None else self._buffer).device

    def _tensors(self):
        return (self._values, self._scales, self._scale) if self._buffer is None else (self._buffer,)

    def _pointers(self):
        """Addresses of the values, the scales and the scale."""
        if self._buffer is None:
            return self._values.data_ptr(), self._scales.data_ptr(), _ptr(self._scale)
        base, at = self._buffer.data_ptr(), self._offsets
        return base, base + at.scales, None if at.scale is None else base + at.scale

    def __repr__(self) -> str:
        return f"Fp4Tensor({self.shape}, {self.format}, {self.device})"


def quantize_fp4(x: torch.Tensor, *, format: str = "nvfp4", scale: torch.Tensor | float | None = None,
                 out: Fp4Tensor | None = None) -> Fp4Tensor:
    """x (..., cols) bf16, fp16 or fp32 with contiguous columns, in 4 bits
    (dgxm_quantize_fp4).  Leading dimensions that do not fold into one stride
    are copied first.

    scale (nvfp4 only): the tensor's scale g as one element of fp32, bf16 or
    fp16 on x's device (what shard.SharedActivationScale returns) or as a
    positive float; None takes amax / 2688 over x, in which a NaN or an
    infinity makes every value NaN.  Block scales are e4m3(amax / (6 g)), codes
    e2m1(x / (s g)); mxfp4: 2^(floor(log2 amax) - 2) and e2m1(x / s).  Every
    rounding is of the real quotient to the nearest, ties to even, saturating;
    a block with a NaN or an infinity reads back as NaN, and so does everything
    under a given g that is NaN, infinite or negative.

    out: an Fp4Tensor of x's shape and the format to write into, its scale
    included."""
    given = scale if isinstance(scale, torch.Tensor) else None
    number = None if scale is None or given is not None else float(scale)
    key = ("q", x.shape, x.stride(), x.dtype, x.get_device(), format, number is not None,
           None if given is None else (given.dtype, given.get_device(), given.numel()),
           None if out is None else (out.shape, out.format, out._devices))

    def make():
        code = _check_format(format)
        _require_cuda(x, given)
        if x.dtype not in _FLOATS:
            raise TypeError(f"x is {x.dtype}: 4-bit quantisation takes bf16, fp16 or fp32")
        if x.ndim < 1 or x.shape[-1] < 1:
            raise ValueError(f"x {tuple(x.shape)} has no columns")
        if x.stride(-1) != 1 and x.shape[-1] > 1:
            raise ValueError("x must have contiguous columns")
        if scale is not None and format == "mxfp4":
            raise ValueError("mxfp4 has no scale for the tensor")
        if given is not None and (given.dtype not in _FLOATS or given.numel() != 1):
            raise ValueError(f"scale {tuple(given.shape)} {given.dtype} is not one element of fp32, bf16 or fp16")
        if out is not None:
            if out.shape != tuple(x.shape) or out.format != format:
                raise ValueError(f"out is {out}, x is {tuple(x.shape)} for {format}")
            _require_cuda(x, *out._tensors())
        desc = _lib.Fp4Desc()
        desc.rows, desc.cols, desc.format = math.prod(x.shape[:-1]), x.shape[-1], code
        desc.dtype = _dtype_code(x.dtype)
        desc.scale_dtype = _lib.DTYPE_F32 if given is None else _dtype_code(given.dtype)
        flat = x.reshape(-1, x.shape[-1]) if x.numel() else x
        folds = x.numel() == 0 or (flat.data_ptr() == x.data_ptr()
                                   and (desc.rows == 1 or flat.stride(0) >= desc.cols))  # not overlapping or expanded
        desc.row_stride = flat.stride(0) if folds and desc.rows > 1 else desc.cols
        need = _lib.load().dgxm_quantize_fp4_workspace() if format == "nvfp4" and scale is None else 0
        return desc, folds, need, _Layout(x.shape, format, x.get_device(), need)

    desc, folds, need, layout = plan(key, make)
    no_graph("", x, given, None if out is None else out._scale)
    if number is not None:  # data, like a scale on the device: checked and set in each call
        if not 0.0 < number < 3.4e38:
            raise ValueError(f"scale {scale} is not a positive finite number")
        desc = _lib.Fp4Desc.from_buffer_copy(desc)  # another thread may be using the plan's own
        desc.scale_value = number
        if desc.scale_value == 0.0:
            raise ValueError(f"scale {scale} is zero in fp32")
    if not folds:
        x = x.reshape(-1, layout.cols).contiguous()
    if out is None:
        buffer = x.new_empty(layout.total, dtype=torch.uint8)
        out = Fp4Tensor._made(buffer, layout)
        work = buffer.data_ptr() + layout.scratch
    else:
        buffer = x.new_empty(need, dtype=torch.uint8) if need else None
        work = _ptr(buffer)
    launch("dgxm_quantize_fp4", layout.devices[0], desc, x.data_ptr(), _ptr(given), *out._pointers(), work, need)
    return out


def dequantize_fp4(t: Fp4Tensor, dtype: torch.dtype = torch.bfloat16, *,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that t stands for, in t.shape and dtype (dgxm_dequantize_fp4):
    code * block scale * scale in fp32, then rounded to dtype.  out: a
    contiguous tensor to write into."""
    key = ("d", t.shape, t.format, dtype, t._devices,
           None if out is None else (out.shape, out.stride(), out.dtype, out.get_device()))

    def make():
        _require_cuda(*t._tensors(), out)
        if dtype not in _FLOATS:
            raise TypeError(f"dtype {dtype} is not bf16, fp16 or fp32")
        if out is not None and (out.shape != t.shape or out.dtype != dtype or not out.is_contiguous()):
            raise ValueError(f"out {tuple(out.shape)} {out.dtype} is not a contiguous {t.shape} {dtype} tensor")
        desc = _lib.Fp4Desc()
        desc.rows, desc.cols, desc.row_stride, desc.format = t.rows, t.cols, t.cols, FORMATS[t.format]
        desc.dtype, desc.scale_dtype = _dtype_code(dtype), _lib.DTYPE_F32
        return desc

    desc = plan(key, make)
    no_graph("", t._scale, out)
    if out is None:
        out = t._tensors()[0].new_empty(t.shape, dtype=dtype)
    launch("dgxm_dequantize_fp4", t._devices[0], desc, *t._pointers(), out.data_ptr())
    return out


def fp4_matmul(a: Fp4Tensor, b: Fp4Tensor, *, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """a (..., k) times the transpose of b (n, k), a Linear's forward
    (dgxm_fp4_matmul): (..., n) in out_dtype (bf16, fp16 or fp32).

    Both operands have one format and share k; bias: (n,) in any of the three
    types.  fp32 accumulation on the block-scaled tensor cores, one rounding.
    out: a tensor of the result's shape and out_dtype to write into, with
    contiguous columns and rows that fold into one stride."""
    key = ("m", a.shape, a.format, a._devices, b.shape, b.format, b._devices, out_dtype,
           None if bias is None else (bias.shape, bias.stride(), bias.dtype, bias.get_device()),
           None if out is None else (out.shape, out.stride(), out.dtype, out.get_device()))

    def make():
        _require_cuda(*a._tensors(), *b._tensors(), bias, out)
        if a.format != b.format:
            raise ValueError(f"a product of {a.format} and {b.format}: both operands have one format")
        if a.cols != b.cols:
            raise ValueError(f"a has {a.cols} columns, b {b.cols}")
        if out_dtype not in _FLOATS:
            raise TypeError(f"out_dtype {out_dtype} is not bf16, fp16 or fp32")
        shape = (*a.shape[:-1], b.rows)
        desc = _lib.Fp4GemmDesc()
        desc.m, desc.n, desc.k, desc.out_stride, desc.format = a.rows, b.rows, a.cols, b.rows, FORMATS[a.format]
        desc.out_dtype = desc.bias_dtype = _dtype_code(out_dtype)
        if bias is not None:
            if bias.dtype not in _FLOATS or tuple(bias.shape) != (b.rows,) or not bias.is_contiguous():
                raise ValueError(f"bias {tuple(bias.shape)} {bias.dtype} is not a contiguous ({b.rows},) vector of "
                                 "bf16, fp16 or fp32")
            desc.bias_dtype = _dtype_code(bias.dtype)
        if out is not None:
            if tuple(out.shape) != shape or out.dtype != out_dtype:
                raise ValueError(f"out {tuple(out.shape)} {out.dtype} is not a {shape} {out_dtype} tensor")
            if out.numel():
                flat = out.reshape(-1, b.rows)
                if (flat.data_ptr() != out.data_ptr() or (b.rows > 1 and flat.stride(1) != 1)
                        or (a.rows > 1 and flat.stride(0) < b.rows)):
                    raise ValueError("out must have contiguous columns and rows that fold into one stride")
                if a.rows > 1:
                    desc.out_stride = flat.stride(0)
        return desc, shape

    desc, shape = plan(key, make)
    no_graph("", bias, a._scale, b._scale, out)
    if out is None:
        out = a._tensors()[0].new_empty(shape, dtype=out_dtype)
    launch("dgxm_fp4_matmul", a._devices[0], desc, *a._pointers(), *b._pointers(), _ptr(bias), out.data_ptr())
    return out

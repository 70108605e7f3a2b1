"""Torch-facing wrappers: a 16-bit Linear with bias, activation, gate and
residual in its epilogue, and its gradients.

The blocks around the attention seam end each branch in such a Linear (inside
the forwards of adapters/flux_family.py:108-265, adapters/krea2.py:130-246 and
adapters/wan_family.py:64-162); fp4.fp4_matmul is its 4-bit sibling.  There is
no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._call import launch, no_graph, plan
from .block_norm import modulation_form
from .ops import _dtype_code, _ptr, _require_cuda
from .qk_norm import _meta

ACTIVATIONS = {"none": _lib.ACT_NONE, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH}
_GRADS = " and take the gradients from linear_backward"


class LinearGrads(NamedTuple):
    """Gradients of linear's arguments, None for those that were None or not wanted."""

    x: torch.Tensor | None
    w: torch.Tensor | None
    bias: torch.Tensor | None
    gate: torch.Tensor | None


def _row_stride(t: torch.Tensor) -> int | None:
    """The one step between the rows of a (rows, cols) or (batch, rows, cols)
    tensor with contiguous columns, or None."""
    cols = t.shape[-1]
    if cols > 1 and t.stride(-1) != 1:
        return None
    lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    if not lead or t.numel() == 0:
        return max(1, cols)
    if len(lead) == 2 and lead[0][1] != lead[1][0] * lead[1][1]:
        return None
    return lead[-1][1] if lead[-1][1] >= cols else None


def _even(t: torch.Tensor | None) -> torch.Tensor | None:
    """t, or a copy whose rows are a step apart."""
    return t if t is None or _row_stride(t) is not None else t.contiguous()


def _check_like(name: str, t: torch.Tensor, shape: tuple, dtypes: tuple) -> None:
    if tuple(t.shape) != shape or t.dtype not in dtypes:
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} is not a {shape} tensor of {' or '.join(map(str, dtypes))}")


def _check_out(name: str, t: torch.Tensor) -> int:
    stride = _row_stride(t)
    if stride is None:
        raise ValueError(f"{name} must have contiguous columns and rows of its own, one step apart")
    return stride


def _describe(x, w, bias, activation, gate) -> _lib.LinearDesc:
    """The checked descriptor of one call without its outputs."""
    _require_cuda(x, w, bias, gate)
    if x.ndim not in (2, 3):
        raise ValueError(f"x must be (rows, k) or (batch, rows, k), got {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x dtype {x.dtype} is not bf16 or fp16")
    if w.ndim != 2 or w.shape[1] != x.shape[-1]:
        raise ValueError(f"w {tuple(w.shape)} is not an (n, {x.shape[-1]}) matrix")
    if w.dtype != x.dtype:
        raise TypeError(f"w is {w.dtype}, x is {x.dtype}: they must share one dtype")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    n, k = w.shape
    if k == 0:
        raise ValueError("a product over no columns")
    desc = _lib.LinearDesc()
    desc.m, desc.n, desc.k = x.shape[:-1].numel(), n, k
    desc.dtype = desc.out_dtype = desc.bias_dtype = desc.gate_dtype = _dtype_code(x.dtype)
    desc.activation = ACTIVATIONS[activation]
    desc.x_stride, desc.w_stride = _row_stride(x) or k, _row_stride(w) or k
    if bias is not None:
        _check_like("bias", bias, (n,), (x.dtype, torch.float32))
        if n > 1 and bias.stride(0) != 1:
            raise ValueError("bias must be contiguous")
        desc.bias_dtype = _dtype_code(bias.dtype)
    if gate is not None:
        b, rows = (1, x.shape[0]) if x.ndim == 2 else x.shape[:2]
        if gate.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"gate is {gate.dtype}, not {x.dtype} or fp32")
        of_rows = gate.unsqueeze(0) if x.ndim == 2 and gate.ndim == 2 and gate.shape[0] == rows else gate
        form, strides = modulation_form("gate", of_rows, b, rows, n)
        if form == _lib.MOD_SAMPLE and rows == 1:
            form = _lib.MOD_TOKEN
        desc.gate_form, desc.sample_rows = form, max(1, rows)
        desc.gate_stride[:] = strides
        desc.gate_dtype = _dtype_code(gate.dtype)
    return desc


def linear(x: torch.Tensor, w: torch.Tensor, *, bias: torch.Tensor | None = None, activation: str = "none",
           gate: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None, return_pre: bool = False):
    """out = residual + gate * act(x w^T + bias) (dgxm_linear), or (out, pre)
    with return_pre, pre = x w^T + bias being what linear_backward takes.

    x (rows, k) or (batch, rows, k) and w (n, k) in bf16 or fp16; bias (n,) and
    gate in x's dtype or fp32; activation "none", "silu", "gelu" or
    "gelu_tanh"; gate (n,), (batch, n), (batch, 1, n) or one value for each
    output ((batch, rows, n), or (rows, n) beside a 2-D x); residual of out's
    shape and dtype; out_dtype x's dtype (the default) or fp32.  fp32
    accumulation and epilogue, one rounding of out and of pre; any sizes, n and
    k up to 2^24.

    out may be residual itself, and must not overlap the inputs in any other
    way.  x, w or residual without contiguous columns and evenly spaced rows is
    copied first, as is x or w whose rows do not lie on 16 bytes.  The same call
    gives the same bits.  No autograd graph is recorded: see linear_backward."""
    return_pre = bool(return_pre)
    key = ("l", _meta(x), _meta(w), _meta(bias), activation, _meta(gate), _meta(residual), out_dtype, _meta(out))

    def make():
        desc = _describe(x, w, bias, activation, gate)
        _require_cuda(x, residual, out)
        shape = (*x.shape[:-1], w.shape[0])
        dtype = out_dtype or (x.dtype if out is None else out.dtype)
        if dtype not in (x.dtype, torch.float32):
            raise TypeError(f"out_dtype {dtype} is not {x.dtype} or fp32")
        desc.out_dtype = _dtype_code(dtype)
        desc.out_stride = desc.pre_stride = desc.residual_stride = max(1, desc.n)
        if out is not None:
            _check_like("out", out, shape, (dtype,))
            desc.out_stride = _check_out("out", out)
        if residual is not None:
            _check_like("residual", residual, shape, (dtype,))
            desc.residual_stride = _row_stride(residual) or max(1, desc.n)
        even = all(t is None or _row_stride(t) is not None for t in (x, w, residual))
        return desc, shape, dtype, even

    desc, shape, dtype, even = plan(key, make)
    no_graph(_GRADS, x, w, bias, gate, residual, out)
    if out is not None and out.numel():
        if out.data_ptr() in (x.data_ptr(), w.data_ptr()):
            raise ValueError("out is the memory of x or w")
        if residual is not None and out.data_ptr() == residual.data_ptr() and out.stride() != residual.stride():
            raise ValueError("out shares the residual's memory with other strides")
    if not even:
        x, w, residual = _even(x), _even(w), _even(residual)
    if out is None:
        out = x.new_empty(shape, dtype=dtype)
    pre = x.new_empty(shape) if return_pre else None
    work, size = _workspace("dgxm_linear_workspace", x, desc, x.data_ptr(), w.data_ptr(),
                            packed=x.data_ptr() % 16 or w.data_ptr() % 16 or desc.x_stride % 8 or desc.w_stride % 8)
    launch("dgxm_linear", x.get_device(), desc, x.data_ptr(), w.data_ptr(), _ptr(bias), _ptr(gate), _ptr(residual),
           out.data_ptr(), _ptr(pre), _ptr(work), size)
    return (out, pre) if return_pre else out


def _workspace(name: str, like: torch.Tensor, desc, *args, packed=True):
    """The workspace that the C function `name` asks for, and its size."""
    size = getattr(_lib.load(), name)(desc, *args) if packed else 0
    if size < 0:
        _lib.check(_lib.DGXM_ERR_INVALID, name)
    return (like.new_empty(size, dtype=torch.uint8) if size else None), size


def linear_backward(dout: torch.Tensor, x: torch.Tensor, w: torch.Tensor, *, bias: torch.Tensor | None = None,
                    activation: str = "none", gate: torch.Tensor | None = None, pre: torch.Tensor | None = None,
                    x_grad: bool = True, w_grad: bool = True) -> LinearGrads:
    """Gradients of linear (dgxm_linear_backward) from the upstream gradient
    dout (x's dtype or fp32), its arguments and pre (needed with an activation
    or a gate); the residual's gradient is dout.

    x_grad, w_grad: whether those are wanted.  They come in x's dtype, bias' and
    gate's in theirs and of their shapes (of bias the shape and dtype alone are
    read).  dz = dout * gate * act'(pre) is rounded to x's dtype for the
    products and not in the sums over rows, which are fp32 in a fixed order:
    the same call gives the same bits.  Inputs without contiguous columns and
    evenly spaced rows are copied first.  w's gradient takes up to 2^24 rows."""
    x_grad, w_grad = bool(x_grad), bool(w_grad)
    key = ("lb", _meta(dout), _meta(x), _meta(w), _meta(bias), activation, _meta(gate), _meta(pre), x_grad, w_grad)

    def make():
        desc = _describe(x, w, bias, activation, gate)
        _require_cuda(x, dout, pre)
        shape = (*x.shape[:-1], w.shape[0])
        _check_like("dout", dout, shape, (x.dtype, torch.float32))
        desc.out_dtype = _dtype_code(dout.dtype)
        desc.out_stride = _row_stride(dout) or max(1, desc.n)
        if pre is not None:
            _check_like("pre", pre, shape, (x.dtype,))
            desc.pre_stride = _row_stride(pre) or max(1, desc.n)
        elif activation != "none" or gate is not None:
            raise ValueError("pre is needed for the gradients of an activation and a gate")
        even = all(t is None or _row_stride(t) is not None for t in (dout, x, w, pre))
        return desc, even

    desc, even = plan(key, make)
    no_graph(_GRADS, dout, x, w, bias, gate, pre)
    if not even:
        dout, x, w, pre = _even(dout), _even(x), _even(w), _even(pre)
    # without rows the sums are of nothing, and the C entry cannot tell of how many samples
    fresh = torch.empty_like if desc.m else torch.zeros_like
    like = lambda t, wanted=True: fresh(t, memory_format=torch.contiguous_format) if wanted and t is not None else None
    grads = LinearGrads(like(x, x_grad), like(w, w_grad), like(bias), like(gate))
    if all(t is None for t in grads):
        return grads
    out = _lib.LinearGradPointers(*map(_ptr, grads))
    work, size = _workspace("dgxm_linear_backward_workspace", x, desc, out, dout.data_ptr(), x.data_ptr(), w.data_ptr())
    launch("dgxm_linear_backward", x.get_device(), desc, out, dout.data_ptr(), x.data_ptr(), w.data_ptr(), _ptr(gate),
           _ptr(pre), _ptr(work), size)
    return grads

"""Torch-facing wrappers: what stands between two branches of a transformer
block, in one pass, and its gradient: the branch joins the residual stream
under a gate (after an RMSNorm of its own, where the block has one), and the
sum is normed and modulated for the next branch.

The blocks around the attention seam do this in five or six elementwise
passes (inside the forwards of adapters/flux_family.py:108-265,
adapters/krea2.py:130-246 and adapters/wan_family.py:64-162).  There is no CPU
path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._call import launch, no_graph, plan
from .ops import _dtype_code, _ptr, _require_cuda
from .qk_norm import _FLOATS, _meta

NORM_NONE, NORM_LAYER, NORM_RMS = _lib.BLOCK_NORM_NONE, _lib.BLOCK_NORM_LAYER, _lib.BLOCK_NORM_RMS
_GRADS = " and take the gradients from block_norm_backward"


class BlockNormGrads(NamedTuple):
    """Gradients of block_norm's arguments, None for those that were None."""

    x: torch.Tensor
    branch: torch.Tensor | None
    gate: torch.Tensor | None
    branch_w: torch.Tensor | None
    norm_w: torch.Tensor | None
    norm_b: torch.Tensor | None
    scale: torch.Tensor | None
    shift: torch.Tensor | None


def _check_like(name: str, t: torch.Tensor, x: torch.Tensor) -> None:
    if t.shape != x.shape or t.dtype != x.dtype:
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} is not a {tuple(x.shape)} {x.dtype} tensor")


def _check_rows(name: str, t: torch.Tensor) -> None:
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous values (its last dimension)")


def _check_out(name: str, t: torch.Tensor, x: torch.Tensor) -> None:
    _check_like(name, t, x)
    _check_rows(name, t)
    if t.numel() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} is an expanded tensor: its rows share memory")


def _strides(t: torch.Tensor) -> list[int]:
    """(batch, row) strides of a (batch, rows, values) tensor."""
    return list(t.stride()[:2])


def modulation_form(name: str, t: torch.Tensor, b: int, rows: int, c: int) -> tuple[int, list[int]]:
    """Whether a modulation of (b, rows, c) tensors holds values for all rows
    ((c), or one sample's for several), each sample ((b, c), (b, 1, c)) or each
    token ((b, rows, c)), and its (batch, row) strides."""
    shape = tuple(t.shape)
    if t.ndim and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous values (its last dimension)")
    if shape in ((c,), (1, c), (1, 1, c)) and (b != 1 or len(shape) == 1):
        return _lib.MOD_SHARED, [0, 0]
    if shape in ((b, c), (b, 1, c)):
        return _lib.MOD_SAMPLE, [t.stride(0), 0]
    if shape == (b, rows, c):
        return _lib.MOD_TOKEN, list(t.stride()[:2])
    raise ValueError(f"{name} {shape} is not ({c},), ({b}, {c}), ({b}, 1, {c}) or ({b}, {rows}, {c})")


def _describe(x, branch, gate, branch_norm, branch_w, norm_mode, norm_w, norm_b, scale, shift, eps) -> _lib.BlockNormDesc:
    """The checked descriptor of one call without its outputs and upstream gradients."""
    _require_cuda(x, branch, gate, branch_w, norm_w, norm_b, scale, shift)
    if x.ndim != 3:
        raise ValueError(f"x must be 3-D (batch, rows, values), got {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"x dtype {x.dtype} is not bf16, fp16 or fp32")
    if norm_mode not in (NORM_NONE, NORM_LAYER, NORM_RMS):
        raise ValueError(f"norm_mode {norm_mode} is not NORM_NONE, NORM_LAYER or NORM_RMS")
    b, rows, c = x.shape
    _check_rows("x", x)
    desc = _lib.BlockNormDesc()
    desc.batch, desc.seq, desc.width = b, rows, c
    desc.dtype = desc.weight_dtype = desc.mod_dtype = _dtype_code(x.dtype)
    desc.norm_mode, desc.branch_norm, desc.eps = norm_mode, int(branch_norm), eps
    desc.x_stride[:] = _strides(x)
    if branch is not None:
        _check_like("branch", branch, x)
        _check_rows("branch", branch)
        desc.branch_stride[:] = _strides(branch)
    elif gate is not None or branch_norm or branch_w is not None:
        raise ValueError("a gate or a branch norm was given without a branch")
    if branch_w is not None and not branch_norm:
        raise ValueError("branch_w was given without branch_norm")
    if norm_mode == NORM_NONE:
        if branch is None:
            raise ValueError("NORM_NONE without a branch leaves nothing to do")
        if any(t is not None for t in (norm_w, norm_b, scale, shift)):
            raise ValueError("norm weights, a scale or a shift were given with NORM_NONE")
    if norm_b is not None and norm_mode == NORM_RMS:
        raise ValueError("norm_b goes with NORM_LAYER")
    weights = [(n, w) for n, w in (("norm_w", norm_w), ("norm_b", norm_b), ("branch_w", branch_w)) if w is not None]
    for name, w in weights:
        if tuple(w.shape) != (c,) or not w.is_contiguous() or w.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} {tuple(w.shape)} {w.dtype} is not a contiguous ({c},) vector of {x.dtype} or fp32")
        if w.dtype != weights[0][1].dtype:
            raise TypeError("norm_w, norm_b and branch_w must share one dtype")
        desc.weight_dtype = _dtype_code(w.dtype)
    mods = [(n, t) for n, t in (("gate", gate), ("scale", scale), ("shift", shift)) if t is not None]
    for name, t in mods:
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} is {t.dtype}, not {x.dtype} or fp32")
        if t.dtype != mods[0][1].dtype:
            raise TypeError("gate, scale and shift must share one dtype")
        desc.mod_dtype = _dtype_code(t.dtype)
        form, strides = modulation_form(name, t, b, rows, c)
        if name == "gate":
            desc.gate_form = form
            desc.gate_stride[:] = strides
            continue
        if name == "shift" and scale is not None and form != desc.mod_form:
            raise ValueError("scale and shift must both be of all rows, of each sample or of each token")
        desc.mod_form = form
        (desc.scale_stride if name == "scale" else desc.shift_stride)[:] = strides
    return desc


def _packed(x: torch.Tensor) -> list[int]:
    return [x.shape[1] * x.shape[2], x.shape[2]]


def _check_memory(name: str, out: torch.Tensor, x: torch.Tensor, branch: torch.Tensor | None) -> None:
    if not x.numel():
        return
    for other in (x, branch):
        if other is not None and out.data_ptr() == other.data_ptr() and out.stride() != other.stride():
            raise ValueError(f"{name} shares its input's memory with other strides")


def block_norm(x: torch.Tensor, branch: torch.Tensor | None = None, *, gate: torch.Tensor | None = None,
               branch_norm: bool = False, branch_w: torch.Tensor | None = None, norm_mode: int = NORM_LAYER,
               norm_w: torch.Tensor | None = None, norm_b: torch.Tensor | None = None,
               scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, eps: float = 1e-6,
               x_out: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Add a branch to the stream x (B, L, C) and norm the sum for the next
    branch (dgxm_block_norm); returns (x_out, out):

        m = branch, or with branch_norm branch / sqrt(mean(branch^2) + eps) * branch_w
        x_out = x + gate * m                     (x itself without a branch)
        out = norm(x_out) * (1 + scale) + shift  (None under NORM_NONE)

    bf16, fp16 or fp32; C up to 8192, any; any strides with contiguous values.
    norm_mode: NORM_LAYER, NORM_RMS or NORM_NONE; norm_w, norm_b (NORM_LAYER)
    and branch_w: (C,) of x's dtype or fp32.  gate, scale and shift, of x's
    dtype or fp32: (C,), (B, C), (B, 1, C), or (B, L, C) with values for each
    token; scale and shift of one form.  Sums are fp32, each output is rounded
    once, and the norm is of the sum before its rounding.  A NaN makes its row's
    norm NaN; an infinity makes NORM_LAYER's row NaN, in NORM_RMS itself NaN and
    the row's other values zero.  Where a row's squares leave fp32's range
    (values above 1e18) its norm is zero, or NaN where its sum does too.

    x_out and out may each be x or branch themselves (same strides); they must
    not overlap the inputs, or each other, in any other way.  No autograd graph
    is recorded: see block_norm_backward."""
    eps, branch_norm = float(eps), bool(branch_norm)  # values, never the identity of a number held in a tensor
    key = ("bn", _meta(x), _meta(branch), _meta(gate), branch_norm, _meta(branch_w), norm_mode, _meta(norm_w),
           _meta(norm_b), _meta(scale), _meta(shift), eps, _meta(x_out), _meta(out))

    def make():
        desc = _describe(x, branch, gate, branch_norm, branch_w, norm_mode, norm_w, norm_b, scale, shift, eps)
        _require_cuda(x, x_out, out)
        if x_out is not None and branch is None:
            raise ValueError("x_out was given without a branch")
        if out is not None and norm_mode == NORM_NONE:
            raise ValueError("out was given with NORM_NONE")
        for name, t, stride in (("x_out", x_out, desc.x_out_stride), ("out", out, desc.out_stride)):
            if t is not None:
                _check_out(name, t, x)
            stride[:] = _packed(x) if t is None else _strides(t)
        return desc

    desc = plan(key, make)
    no_graph(_GRADS, x, branch, gate, branch_w, norm_w, norm_b, scale, shift, x_out, out)
    if branch is not None:
        if x_out is None:
            x_out = torch.empty_like(x, memory_format=torch.contiguous_format)
        else:
            _check_memory("x_out", x_out, x, branch)
    if norm_mode != NORM_NONE:
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        else:
            _check_memory("out", out, x, branch)
            if x_out is not None and x.numel() and out.data_ptr() == x_out.data_ptr():
                raise ValueError("x_out and out share their memory")
    launch("dgxm_block_norm", x.get_device(), desc, x.data_ptr(), _ptr(branch), _ptr(gate), _ptr(scale), _ptr(shift),
           _ptr(norm_w), _ptr(norm_b), _ptr(branch_w), _ptr(x_out), _ptr(out))
    return x if branch is None else x_out, out


def block_norm_backward(dy: torch.Tensor | None, dx_out: torch.Tensor | None, x_out: torch.Tensor,
                        branch: torch.Tensor | None = None, *, gate: torch.Tensor | None = None,
                        branch_norm: bool = False, branch_w: torch.Tensor | None = None, norm_mode: int = NORM_LAYER,
                        norm_w: torch.Tensor | None = None, norm_b: torch.Tensor | None = None,
                        scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
                        eps: float = 1e-6) -> BlockNormGrads:
    """Gradients of block_norm (dgxm_block_norm_backward) from the upstream
    gradients dy of its out (None under NORM_NONE) and dx_out of its x_out
    (None where nothing else uses it), its x_out (without a branch: its x) and
    its other arguments.

    dy and dx_out may have any strides: one without contiguous values (the
    expanded ones that a sum passes back) is copied first.  Gradients have the
    shapes and dtypes of what they belong to, sums over rows are fp32 in a
    fixed order: the same call gives the same bits.  Without a gate and a
    branch norm the branch's gradient is x's, and under NORM_NONE x's is dx_out: those are
    returned as one tensor."""
    eps, branch_norm = float(eps), bool(branch_norm)
    key = ("bb", _meta(dy), _meta(dx_out), _meta(x_out), _meta(branch), _meta(gate), branch_norm, _meta(branch_w),
           norm_mode, _meta(norm_w), _meta(norm_b), _meta(scale), _meta(shift), eps)

    def make():
        x = x_out
        desc = _describe(x, branch, gate, branch_norm, branch_w, norm_mode, norm_w, norm_b, scale, shift, eps)
        _require_cuda(x, dy, dx_out)
        if (dy is None) != (norm_mode == NORM_NONE):
            raise ValueError("dy comes with a norm, and only then")
        if dy is None and dx_out is None:
            raise ValueError("neither dy nor dx_out was given")
        for name, t, stride in (("dy", dy, desc.dy_stride), ("dx_out", dx_out, desc.dx_out_stride)):
            if t is not None:
                _check_like(name, t, x)
                stride[:] = _strides(t) if t.stride(2) == 1 or t.shape[2] == 1 else _packed(x)
        desc.x_out_stride[:] = desc.out_stride[:] = _packed(x)
        need = _lib.load().dgxm_block_norm_backward_workspace(desc)
        if need < 0:
            _lib.check(_lib.DGXM_ERR_INVALID, "dgxm_block_norm_backward_workspace")
        scattered = [t is not None and t.shape[2] > 1 and t.stride(2) != 1 for t in (dy, dx_out)]
        summed = (any(w is not None for w in (norm_w, norm_b, branch_w)) or (gate is not None and desc.gate_form != _lib.MOD_TOKEN)
                  or ((scale is not None or shift is not None) and desc.mod_form != _lib.MOD_TOKEN))
        return desc, need if summed else 0, scattered

    desc, need, scattered = plan(key, make)
    no_graph(_GRADS, dy, dx_out, x_out, branch, gate, branch_w, norm_w, norm_b, scale, shift)
    if scattered[0]:
        dy = dy.contiguous()
    if scattered[1]:
        dx_out = dx_out.contiguous()
    like = lambda t: None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)
    apart = branch is not None and (gate is not None or branch_norm)
    gx = dx_out if norm_mode == NORM_NONE else like(x_out)
    gbranch = like(branch) if apart else gx if branch is not None else None
    grads = BlockNormGrads(gx, gbranch, like(gate), like(branch_w), like(norm_w), like(norm_b), like(scale), like(shift))
    if norm_mode == NORM_NONE and not apart:
        return grads
    work = x_out.new_empty(need, dtype=torch.uint8) if need else None
    out = _lib.BlockNormGradPointers(None if norm_mode == NORM_NONE else gx.data_ptr(), gbranch.data_ptr() if apart else None,
                                     _ptr(grads.gate), _ptr(grads.scale), _ptr(grads.shift), _ptr(grads.norm_w),
                                     _ptr(grads.norm_b), _ptr(grads.branch_w))
    launch("dgxm_block_norm_backward", x_out.get_device(), desc, out, _ptr(dy), _ptr(dx_out), x_out.data_ptr(),
           branch.data_ptr() if apart else None, _ptr(gate), _ptr(scale), _ptr(norm_w), _ptr(norm_b), _ptr(branch_w),
           _ptr(work), need)
    return grads

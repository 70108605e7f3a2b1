"""Torch-facing wrappers: RMSNorm of each query and key head with the rotary
position embedding in the same pass, on this rank's own tensors, and its
gradient.

The norm is the QKNorm of the Flux and Krea2 blocks, over each head's values,
which those blocks run with RoPE before the attention seam (inside the forwards
of adapters/flux_family.py:108-265 and adapters/krea2.py:130-246).  Wan's
norm_q / norm_k go over all heads of a row (adapters/wan_family.py:70-71) and
are not this norm; its rotation (adapters/wan_family.py:73) is NORM_NONE here.
prologue.py fuses both norms with the Ulysses scatter; the calls here serve
where nothing is scattered (one rank, ring attention, cross attention) and
where the block is trained.  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from ._call import launch, no_graph, plan
from .ops import _dtype_code, _ptr, _require_cuda

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_GRADS = " and take the gradients from qk_norm_rope_backward"


def _check_rows(name: str, t: torch.Tensor, q: torch.Tensor, whole: bool = True) -> None:
    if t.ndim != 4:
        raise ValueError(f"{name} must be 4-D (batch, rows, heads, head_dim), got {tuple(t.shape)}")
    if t.shape[:2] != q.shape[:2] or t.shape[3] != q.shape[3]:
        raise ValueError(f"{name} {tuple(t.shape)} does not share (batch, rows, head_dim) with q {tuple(q.shape)}")
    if t.dtype != q.dtype:
        raise TypeError(f"{name} is {t.dtype}, q is {q.dtype}: they must share one dtype")
    if whole and t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name} must have a contiguous head_dim")


def _check_out(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.shape != like.shape or t.dtype != like.dtype or t.stride(3) != 1:
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} is not a {tuple(like.shape)} {like.dtype} tensor with "
                         "contiguous head_dim")
    if t.numel() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} is an expanded tensor: its rows share memory")


def _check_in_place(name: str, out: torch.Tensor, src: torch.Tensor, other: torch.Tensor | None) -> None:
    if src.numel() == 0:
        return
    if out.data_ptr() == src.data_ptr() and out.stride() != src.stride():
        raise ValueError(f"{name} shares its input's memory with other strides")
    if other is not None and other.numel() and out.data_ptr() == other.data_ptr():
        raise ValueError(f"{name} is the memory of the other tensor")


def _describe(q, k, norm_mode, wq, wk, eps, rope, rope_halves) -> _lib.QkNormDesc:
    """The checked descriptor of one call without its output and gradient strides."""
    _require_cuda(q, k, wq, wk, rope)
    if q.dtype not in _FLOATS:
        raise TypeError(f"q/k dtype {q.dtype} is not bf16, fp16 or fp32")
    _check_rows("q", q, q)
    if k is not None:
        _check_rows("k", k, q)
    b, l, hq, d = q.shape
    desc = _lib.QkNormDesc()
    desc.batch, desc.seq, desc.q_heads, desc.k_heads, desc.head_dim = b, l, hq, 0 if k is None else k.shape[2], d
    desc.dtype = desc.weight_dtype = _dtype_code(q.dtype)
    desc.norm_mode, desc.rope_halves, desc.eps = norm_mode, int(rope_halves), eps
    desc.q_stride[:] = q.stride()[:3]
    if k is not None:
        desc.k_stride[:] = k.stride()[:3]
    weights = [(n, w) for n, w in (("norm_q_w", wq), ("norm_k_w", wk)) if w is not None]
    if weights and norm_mode == _lib.NORM_NONE:
        raise ValueError("norm weights were given with norm_mode NORM_NONE")
    if k is not None and (wq is None) != (wk is None):
        raise ValueError("give both norm weights or neither")
    if k is None and wk is not None:
        raise ValueError("norm_k_w was given without k")
    for name, w in weights:
        if tuple(w.shape) != (d,) or not w.is_contiguous() or w.dtype not in (q.dtype, torch.float32):
            raise ValueError(f"{name} {tuple(w.shape)} {w.dtype} is not a contiguous ({d},) vector of {q.dtype} or fp32")
        if w.dtype != weights[0][1].dtype:
            raise TypeError("norm_q_w and norm_k_w must share one dtype")
        desc.weight_dtype = _dtype_code(w.dtype)
    if rope is not None:
        if (rope.dtype != torch.float32 or rope.ndim not in (3, 4) or rope.shape[-1] != 2 or rope.shape[-3] != l
                or (rope.ndim == 4 and rope.shape[0] != b) or not rope.is_contiguous()):
            raise ValueError(f"rope {tuple(rope.shape)} {rope.dtype} is not a contiguous fp32 ({l}, pairs, 2) or "
                             f"({b}, {l}, pairs, 2) table")
        desc.rot_dim = 2 * rope.shape[-2]
        desc.rope_batch_stride = 0 if rope.ndim == 3 else rope.stride(0)
        if desc.rot_dim > d:
            raise ValueError(f"rope has {rope.shape[-2]} pairs for a head_dim of {d}")
    return desc


def _meta(t: torch.Tensor | None):
    """What the checks and the descriptor of a call read of a tensor."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None = None, *, norm_mode: int = _lib.NORM_HEAD,
                 norm_q_w: torch.Tensor | None = None, norm_k_w: torch.Tensor | None = None, eps: float = 1e-6,
                 rope: torch.Tensor | None = None, rope_halves: bool = False, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMSNorm each head of q (B, L, Hq, D) and k (B, L, Hk, D) and rotate it
    by its token's angles (dgxm_qk_norm_rope); returns (q_out, k_out).

    bf16, fp16 or fp32; D a multiple of 8 up to 256; any strides with a
    contiguous D (slices of one QKV projection, expanded tensors); k may be
    None or have fewer heads.  norm_q_w / norm_k_w: (D,) in q's dtype or fp32.
    rope: fp32 (L, P, 2) or (B, L, P, 2) cosines and sines of P <= D / 2 pairs
    (prologue.rope_table); the first 2 P values of a head are rotated, values
    2i and 2i + 1 with each other, or i and P + i with rope_halves.  norm_mode
    NORM_NONE rotates alone.  Sums and rotation are fp32, rounded once; a head
    whose sum of squares leaves fp32's range comes out zero (values above 1e18)
    or, with an eps of zero, loses digits and ends infinite or NaN (values below
    1e-18).

    q_out / k_out may be q / k themselves (same strides); they must not
    overlap the inputs, or each other, in any other way.  No autograd graph is recorded: see
    qk_norm_rope_backward."""
    eps, rope_halves = float(eps), bool(rope_halves)  # values, never the identity of a number held in a tensor
    key = ("f", _meta(q), _meta(k), norm_mode, _meta(norm_q_w), _meta(norm_k_w), eps, _meta(rope), rope_halves,
           _meta(q_out), _meta(k_out))

    def make():
        desc = _describe(q, k, norm_mode, norm_q_w, norm_k_w, eps, rope, rope_halves)
        _require_cuda(q, q_out, k_out)
        if k is None and k_out is not None:
            raise ValueError("k_out was given without k")
        for out, src, stride, name in ((q_out, q, desc.q_out_stride, "q_out"), (k_out, k, desc.k_out_stride, "k_out")):
            if out is not None:
                _check_out(name, out, src)
                stride[:] = out.stride()[:3]
            elif src is not None:
                h, d = src.shape[2], src.shape[3]
                stride[:] = [src.shape[1] * h * d, h * d, d]
        return desc

    desc = plan(key, make)
    no_graph(_GRADS, q, k, norm_q_w, norm_k_w, rope, q_out, k_out)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_in_place("q_out", q_out, q, k)
    if k is not None:
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        else:
            _check_in_place("k_out", k_out, k, q)
            if k_out.data_ptr() == q_out.data_ptr() and k.numel() and q.numel():
                raise ValueError("q_out and k_out share their memory")
    launch("dgxm_qk_norm_rope", q.get_device(), desc, q.data_ptr(), _ptr(k), _ptr(norm_q_w), _ptr(norm_k_w),
           _ptr(rope), q_out.data_ptr(), _ptr(k_out))
    return q_out, k_out


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor | None = None,
                          *, norm_mode: int = _lib.NORM_HEAD, norm_q_w: torch.Tensor | None = None,
                          norm_k_w: torch.Tensor | None = None, eps: float = 1e-6,
                          rope: torch.Tensor | None = None, rope_halves: bool = False):
    """Gradients of qk_norm_rope (dgxm_qk_norm_rope_backward): (gq, gk, gwq,
    gwk) from the upstream gradients dq, dk of its outputs and its inputs.

    dq and dk may have any strides: one without a contiguous D (the expanded
    ones that a sum passes back) is copied first, unlike q and k.  gq and gk
    have the full shape of q and k (an expanded input's gradient is
    the caller's to sum) and gwq / gwk the weights' dtype, each summed over
    batch, rows and heads in fp32; gk, gwq and gwk are None where the
    corresponding argument is.  A weight that serves both q and k has the sum
    of gwq and gwk as its gradient.  The sums' order is fixed: the same call
    gives the same bits."""
    eps, rope_halves = float(eps), bool(rope_halves)
    key = ("b", _meta(dq), _meta(dk), _meta(q), _meta(k), norm_mode, _meta(norm_q_w), _meta(norm_k_w), eps,
           _meta(rope), rope_halves)

    def make():
        desc = _describe(q, k, norm_mode, norm_q_w, norm_k_w, eps, rope, rope_halves)
        _require_cuda(q, dq, dk)
        if (dk is None) != (k is None):
            raise ValueError("dk and k come together")
        for up, src, ups, outs, name in ((dq, q, desc.dq_stride, desc.q_out_stride, "dq"),
                                         (dk, k, desc.dk_stride, desc.k_out_stride, "dk")):
            if src is None:
                continue
            _check_rows(name, up, q, whole=False)
            if up.shape != src.shape:
                raise ValueError(f"{name} {tuple(up.shape)} is not the gradient of a {tuple(src.shape)} tensor")
            h, d = src.shape[2], src.shape[3]
            outs[:] = [src.shape[1] * h * d, h * d, d]
            ups[:] = outs if up.stride(3) != 1 else up.stride()[:3]
        need = _lib.load().dgxm_qk_norm_rope_backward_workspace(desc)
        if need < 0:
            _lib.check(_lib.DGXM_ERR_INVALID, "dgxm_qk_norm_rope_backward_workspace")
        scattered = dq.stride(3) != 1 or (dk is not None and dk.stride(3) != 1)
        return desc, need, scattered

    desc, need, scattered = plan(key, make)
    no_graph(_GRADS, dq, dk, q, k, norm_q_w, norm_k_w, rope)
    if scattered:
        dq = dq if dq.stride(3) == 1 else dq.contiguous()
        dk = dk if dk is None or dk.stride(3) == 1 else dk.contiguous()
    gq = torch.empty_like(q, memory_format=torch.contiguous_format)
    gk = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    gwq = None if norm_q_w is None else torch.empty_like(norm_q_w)
    gwk = None if norm_k_w is None else torch.empty_like(norm_k_w)
    work = q.new_empty(need, dtype=torch.uint8) if need and gwq is not None else None
    launch("dgxm_qk_norm_rope_backward", q.get_device(), desc, dq.data_ptr(), _ptr(dk), q.data_ptr(), _ptr(k),
           _ptr(norm_q_w), _ptr(norm_k_w), _ptr(rope), gq.data_ptr(), _ptr(gk), _ptr(gwq), _ptr(gwk), _ptr(work),
           need if work is not None else 0)
    return gq, gk, gwq, gwk

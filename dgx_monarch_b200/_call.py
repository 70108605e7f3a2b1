"""The short path of a call whose arguments have been seen before.

A small operator's kernel runs for a few microseconds, as long as Python
takes for a few attribute reads, so the wrappers check a call's arguments
once for each combination of sizes, strides, types and devices, keep the C
descriptor that came of it (never data or an address), and launch on the raw
handle of the current stream.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

_PLANS: dict = {}
_MOST_PLANS = 512
_FUNCS: dict = {}


def plan(key, make):
    """The plan of `key`, made (and its arguments checked) on first sight."""
    found = _PLANS.get(key)
    if found is None:
        found = make()
        if len(_PLANS) >= _MOST_PLANS:
            _PLANS.clear()
        _PLANS[key] = found
    return found


def launch(name: str, index: int, *args) -> None:
    """Call the C entry `name` with args and the current stream of CUDA device
    `index`, on that device; raise on a status."""
    fn = _FUNCS.get(name)
    if fn is None:
        fn = _FUNCS[name] = getattr(_lib.load(), name)
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def no_graph(where: str, *tensors: torch.Tensor | None) -> None:
    """Refuse tensors whose gradient the caller expects autograd to follow, in
    reverse or (under a dual level only, and whether or not reverse mode is on)
    forward mode."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the B200 kernels record no autograd graph: call them under torch.no_grad()" + where)
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the B200 kernels carry no forward-mode tangent: pass the primal of a dual tensor")

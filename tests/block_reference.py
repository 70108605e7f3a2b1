"""The operators between two branches of a block in 64 bits, with the error
that fp32 arithmetic and one rounding of each output may leave.

A sum of C values in a block passes at most 16 additions of one thread, 5 of
its warp and 5 across warps; SUM = 32 roundings cover those and the product.
rsqrt is off by 2 ulp and its argument by a few roundings: ROOT = 8.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24  # half a step of fp32, relative
SUM, ROOT = 32 * U, 8 * U


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half a step below the type's normal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def lift(t, rows: int):
    """A modulation against (batch, rows, values) in 64 bits."""
    if t is None:
        return None
    t = t.double()
    if t.ndim == 1:
        return t[None, None]
    return t[:, None] if t.ndim == 2 else t


def _mean(t):
    return t.mean(-1, keepdim=True)


def _rms(t):
    return (t * t).mean(-1, keepdim=True).sqrt()


def forward(x, branch=None, *, gate=None, branch_norm=False, branch_w=None, mode="layer", norm_w=None, norm_b=None,
            scale=None, shift=None, eps=1e-6):
    """(x_out, out) and the bounds of their errors before rounding."""
    r = x.double()
    size = r.abs()  # what r's roundings are relative to
    rows = x.shape[1]
    if branch is not None:
        m = branch.double()
        rel = 0.0
        if branch_norm:
            m = m / (_mean(m * m) + eps).sqrt()
            rel = SUM + ROOT
            if branch_w is not None:
                m = m * branch_w.double()
        g = lift(gate, rows)
        m = m if g is None else m * g
        r = r + m
        size = size + m.abs()
        r_err = 4 * U * size + rel * m.abs()
    else:
        r_err = torch.zeros_like(r)
    if mode == "none":
        return r, None, r_err, None
    if mode == "layer":
        mean = _mean(r)
        mean_err = SUM * _mean(r.abs()) + _mean(r_err)
        dev, dev_err = r - mean, r_err + mean_err + U * (r.abs() + mean.abs())
    else:
        dev, dev_err = r, r_err
    k = 1 / (_mean(dev * dev) + eps).sqrt()
    root_rel = SUM + ROOT + k * _rms(dev_err)
    n = dev * k
    n_err = dev_err * k + n.abs() * root_rel
    up = 1.0 if scale is None else 1 + lift(scale, rows)
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if norm_w is None else norm_w.double()
    h = n * w
    y, parts = h * up, (h * up).abs()
    err = n_err * (w * up).abs()
    if norm_b is not None:
        y, parts = y + norm_b.double() * up, parts + (norm_b.double() * up).abs()
    if shift is not None:
        y, parts = y + lift(shift, rows), parts + lift(shift, rows).abs()
    return r, y, r_err, err + 8 * U * parts


def _reduce(values, like):
    """Sum (batch, rows, values) to the shape of a modulation."""
    if like.ndim == 3 and like.shape[1] == values.shape[1] and like.shape[0] == values.shape[0]:
        return values
    if like.shape[-1] == like.numel():
        return values.sum((0, 1)).view(like.shape)
    return values.sum(1).view(like.shape)


def backward(dy, dr, r, branch=None, *, gate=None, branch_norm=False, branch_w=None, mode="layer", norm_w=None, norm_b=None,
             scale=None, shift=None, eps=1e-6):
    """{name: (gradient, bound of its error before rounding)}."""
    b, rows, c = r.shape
    depth = (b * rows + 64) * U  # a sum over rows, in whatever order
    got = {}
    big = torch.zeros(b, rows, c, dtype=torch.float64, device=r.device) if dr is None else dr.double()
    big_err = torch.zeros_like(big)
    one = torch.ones(c, dtype=torch.float64, device=r.device)
    if mode != "none":
        r, dy = r.double(), dy.double()
        dev, dev_err = r, torch.zeros_like(r)
        if mode == "layer":
            mean = _mean(r)
            dev, dev_err = r - mean, SUM * _mean(r.abs()) + U * (r.abs() + mean.abs())
        k = 1 / (_mean(dev * dev) + eps).sqrt()
        k_rel = SUM + ROOT + k * _rms(dev_err)
        n = dev * k
        n_err = dev_err * k + n.abs() * (k_rel + U)
        w = one if norm_w is None else norm_w.double()
        bias = 0 * one if norm_b is None else norm_b.double()
        up = 1 + lift(scale, rows) if scale is not None else one
        h, e = n * w + bias, dy * up
        for name, like, value, err in (("scale", scale, dy * h, dy.abs() * (n_err * w.abs() + 4 * U * (n * w).abs() + 4 * U * bias.abs())),
                                       ("shift", shift, dy, 0 * dy),
                                       ("norm_w", norm_w, e * n, e.abs() * (n_err + 4 * U * n.abs())),
                                       ("norm_b", norm_b, e, 4 * U * e.abs())):
            if like is not None:
                # the kernel's sums of a sample are multiplied once more: 4 roundings
                got[name] = (_reduce(value, like), _reduce(err + (depth + 4 * U) * (dy.abs() * (n * w).abs() + dy.abs() * bias.abs() if name == "scale" else value.abs()), like))
        dn = e * w
        m2, m2_err = _mean(dn * n), SUM * _mean((dn * n).abs()) + _mean(dn.abs() * n_err) + 4 * U * _mean((dn * n).abs())
        m1, m1_err = (_mean(dn), (SUM + 4 * U) * _mean(dn.abs())) if mode == "layer" else (0 * m2, 0 * m2)
        inner = dn - m1 - n * m2
        inner_err = 6 * U * (dn.abs() + m1.abs() + (n * m2).abs()) + m1_err + n_err * m2.abs() + n.abs() * m2_err
        big_err = k * (inner_err + inner.abs() * k_rel) + 2 * U * (big.abs() + (k * inner).abs())
        big = big + k * inner
    got["x"] = (big, big_err)
    if branch is None:
        return got
    m, m_rel = branch.double(), 0.0
    k2, w2 = None, one if branch_w is None else branch_w.double()
    if branch_norm:
        k2 = 1 / (_mean(m * m) + eps).sqrt()
        m, m_rel = m * k2, SUM + ROOT + U
    g = lift(gate, rows) if gate is not None else one
    dm, dm_err = big * g, (big_err + 2 * U * big.abs()) * g.abs()
    if gate is not None:
        value = big * m * w2
        err = big_err * (m * w2).abs() + (m_rel + 6 * U) * value.abs()
        got["gate"] = (_reduce(value, gate), _reduce(err + depth * value.abs(), gate))
    if branch_norm:
        if branch_w is not None:
            value = dm * m
            got["branch_w"] = (_reduce(value, branch_w), _reduce(dm_err * m.abs() + (m_rel + 6 * U + depth) * value.abs(), branch_w))
        dn2, dn2_err = dm * w2, (dm_err + U * dm.abs()) * w2.abs()
        m3 = _mean(dn2 * m)
        m3_err = _mean(dn2_err * m.abs()) + (SUM + m_rel + 2 * U) * _mean((dn2 * m).abs())
        inner = dn2 - m * m3
        err = dn2_err + m.abs() * m3_err + (m * m3).abs() * (m_rel + 4 * U) + 4 * U * dn2.abs()
        dm, dm_err = k2 * inner, k2 * (err + inner.abs() * (SUM + ROOT))
    got["branch"] = (dm, dm_err)
    return got


def check(name, got, want, err):
    """got, rounded once to its type, against want with a bound of the error before rounding."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    half = half_step(got.dtype)
    limit = half * want.abs() + (1 + half) * err + tiny(got.dtype)
    over = (got.double() - want).abs() - limit
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{name}: {worst} beyond the limit at {tuple(int(i) for i in (over == over.max()).nonzero()[0])}"

"""Per-head Q/K RMSNorm with the rotary embedding, and its gradient, against
the formulas in 64 bits.

Tolerances.  The kernels compute in fp32 and round once, so an output is off
by at most half a step of its type, eps / 2 relative, plus the fp32 error.  A
row's sum of squares takes 8 additions in a lane and at most 5 across lanes
(13 * 2^-24 relative, halved by the root), rsqrt 2 steps (2^-22) and the
products and the rotation under 6 roundings (2^-21.4): below 2^-20 of the
terms' magnitudes.  The gradient adds one more such sum and product: 2^-19.
A weight's gradient sums its rows in fp32; no addition chain here is longer
than 256, hence 256 * 2^-24 = 2^-16 of the sum of magnitudes.
"""
from __future__ import annotations

import pytest
import torch

from dgx_monarch_b200 import _lib
from dgx_monarch_b200.qk_norm import qk_norm_rope, qk_norm_rope_backward

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _table(l, pairs, g, batch=None):
    shape = (l, pairs) if batch is None else (batch, l, pairs)
    ang = 40 * torch.rand(*shape, device="cuda", generator=g, dtype=torch.float64)
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def _partner(x, rot, halves):
    """For each value of the last axis the one it is rotated with (itself past rot)."""
    z, rest = x[..., :rot], x[..., rot:]
    if halves:
        z = torch.cat([z[..., rot // 2:], z[..., :rot // 2]], -1)
    else:
        z = z.unflatten(-1, (rot // 2, 2)).flip(-1).flatten(-2)
    return torch.cat([z, rest], -1)


def _turn(x, rope, halves, sign=1):
    """(rotated x, sum of the magnitudes of its terms), 64 bits."""
    if rope is None:
        return x, x.abs()
    rot = 2 * rope.shape[-2]
    t = rope.double()
    if t.ndim == 3:
        t = t[None]
    c, s = t[..., 0][:, :, None], sign * t[..., 1][:, :, None]
    if halves:
        c, s = torch.cat([c, c], -1), torch.cat([-s, s], -1)
    else:
        c, s = c.repeat_interleave(2, -1), torch.stack([-s, s], -1).flatten(-2)
    p = _partner(x, rot, halves)
    y = torch.cat([x[..., :rot] * c + p[..., :rot] * s, x[..., rot:]], -1)
    return y, x.abs() + p.abs()


def _close(got, want, fp32_error):
    assert got.shape == want.shape
    eps = torch.finfo(got.dtype).eps
    tol = eps / 2 * 1.001 * want.abs() + fp32_error + torch.finfo(got.dtype).tiny * eps
    bad = (got.double() - want).abs() > tol
    assert torch.isfinite(got).all()
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


def _check_forward(got, x, w, rope, halves, eps, norm):
    v = x.double()
    if norm:
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * (1 if w is None else w.double())
    want, size = _turn(v, rope, halves)
    _close(got, want, 2.0 ** -20 * size)


def _check_backward(gx, gw, dy, x, w, rope, halves, eps, norm):
    g, size = _turn(dy.double(), rope, halves, -1)
    if not norm:
        _close(gx, g, 2.0 ** -20 * size)
        return
    v = x.double()
    r = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    n = v * r
    if gw is not None:
        _close(gw, (g * n).sum((0, 1, 2)), 2.0 ** -16 * (size * n.abs()).sum((0, 1, 2)))
    wd = 1 if w is None else w.double()
    want = r * (g * wd - n * (g * wd * n).mean(-1, keepdim=True))
    mag = r * (size * abs(wd) + n.abs() * (size * abs(wd) * n.abs()).mean(-1, keepdim=True))
    _close(gx, want, 2.0 ** -19 * mag)


CASES = [
    # batch, rows, q heads, k heads, dim, rot, halves, norm, weights' dtype, dtype, table per batch item
    (1, 1, 1, 1, 8, 8, False, True, None, BF16, False),
    (1, 1, 40, 40, 128, 128, False, True, BF16, BF16, False),
    (2, 33, 5, 1, 128, 128, True, True, BF16, BF16, True),
    (3, 7, 12, 3, 64, 64, False, True, F32, BF16, False),
    (1, 129, 9, 9, 96, 64, True, True, F16, F16, False),
    (2, 17, 4, 2, 72, 36, True, True, F16, F16, False),      # halves of 18: partners off the lanes' vectors
    (2, 17, 4, 2, 72, 36, False, True, F32, F16, False),
    (1, 65, 6, 6, 256, 256, True, True, F32, F32, False),
    (1, 31, 3, 2, 256, 20, True, True, F32, F32, True),
    (4, 5, 2, 2, 40, 2, False, True, None, F32, False),
    (1, 50, 17, 4, 128, 0, False, True, BF16, BF16, False),  # norm alone
    (2, 21, 8, 2, 128, 128, False, False, None, BF16, False),  # rotation alone
    (2, 21, 8, 2, 80, 40, True, False, None, F16, False),
    (1, 11, 2, 2, 24, 0, False, False, None, F32, False),    # neither
]


@pytest.mark.parametrize("b,l,hq,hk,d,rot,halves,norm,wt,dtype,per_item", CASES)
def test_forward_and_gradient(b, l, hq, hk, d, rot, halves, norm, wt, dtype, per_item):
    g = _gen(l)
    # slices of one projection's output, v between
    qkv = (torch.randn(b, l, hq + 2 * hk, d, device="cuda", generator=g)
           * torch.exp(torch.randn(b, l, 1, 1, device="cuda", generator=g))).to(dtype)
    q, k = qkv[:, :, :hq], qkv[:, :, hq + hk:]
    wq = wk = None
    if wt is not None:
        wq, wk = (torch.randn(d, device="cuda", generator=g).to(wt) for _ in range(2))
    rope = _table(l, rot // 2, g, b if per_item else None) if rot else None
    how = {"norm_mode": _lib.NORM_HEAD if norm else _lib.NORM_NONE, "norm_q_w": wq, "norm_k_w": wk, "eps": 1e-5,
           "rope": rope, "rope_halves": halves}
    before = qkv.clone()
    yq, yk = qk_norm_rope(q, k, **how)
    assert yq.dtype == dtype and yq.is_contiguous() and yk.is_contiguous()
    _check_forward(yq, q, wq, rope, halves, 1e-5, norm)
    _check_forward(yk, k, wk, rope, halves, 1e-5, norm)
    dq, dk = (torch.randn(b, l, h, d, device="cuda", generator=g).to(dtype) for h in (hq, hk))
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, **how)
    assert (gwq is None) == (wt is None) and (gwk is None) == (wt is None)
    _check_backward(gq, gwq, dq, q, wq, rope, halves, 1e-5, norm)
    _check_backward(gk, gwk, dk, k, wk, rope, halves, 1e-5, norm)
    assert torch.equal(qkv, before)
    again = qk_norm_rope_backward(dq, dk, q, k, **how)
    for x, y in zip((gq, gk, gwq, gwk), again):
        assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("halves", [False, True])
def test_odd_alignment_and_transposed_strides(dtype, halves):
    """Bases and strides off 16 bytes, and (B, H, L, D) storage."""
    g = _gen(3)
    b, l, h, d = 2, 19, 3, 64
    flat = torch.randn(b * l * h * (d + 1) + 1, device="cuda", generator=g).to(dtype)
    q = flat[1:].view(b, l, h, d + 1)[..., :d]
    k = torch.randn(b, h, l, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
    wq = torch.randn(d + 1, device="cuda", generator=g).to(dtype)[1:]
    wk = torch.randn(d, device="cuda", generator=g).to(dtype)
    rope = _table(l, d // 2 + 1, g)[:, 1:].contiguous()
    off = torch.empty(rope.numel() + 1, device="cuda")
    off[1:] = rope.flatten()
    rope = off[1:].view(rope.shape)  # a table that starts 4 bytes into its storage
    out = torch.full((b, l, h, d + 3), 7.0, device="cuda").to(dtype)
    yq, yk = qk_norm_rope(q, k, norm_q_w=wq, norm_k_w=wk, rope=rope, rope_halves=halves, q_out=out[..., 1:d + 1])
    assert yq.data_ptr() == out[..., 1:].data_ptr()
    assert (out[..., 0] == 7).all() and (out[..., d + 1:] == 7).all()
    _check_forward(yq, q, wq, rope, halves, 1e-6, True)
    _check_forward(yk, k, wk, rope, halves, 1e-6, True)
    dq = torch.randn(b, h, l, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
    dk = torch.randn(b, l, h, d + 1, device="cuda", generator=g).to(dtype)[..., 1:]
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, norm_q_w=wq, norm_k_w=wk, rope=rope, rope_halves=halves)
    _check_backward(gq, gwq, dq, q, wq, rope, halves, 1e-6, True)
    _check_backward(gk, gwk, dk, k, wk, rope, halves, 1e-6, True)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("b,l,hq,hk,d,rot,dtype,pad", [
    (1, 4000, 20, 4, 96, 96, F16, 0),    # two chunks of five rows a lane group, and one that two rows fill
    (1, 4000, 13, 3, 128, 128, BF16, 0),  # seven rows, six in the other lane group
    (2, 2000, 13, 3, 128, 64, F32, 0),   # a full ring of four, the last chunk shorter
    (1, 4001, 30, 10, 64, 64, BF16, 0),  # a full ring of eight, four lane groups
    (4, 1000, 5, 2, 256, 256, BF16, 0),  # one lane group
    (2, 2000, 13, 3, 72, 36, F16, 0),    # halves off the lanes' vectors
    (1, 4000, 13, 3, 96, 96, BF16, 1),   # rows off 16 bytes
    (1, 4001, 13, 3, 96, 36, F32, 1),
])
def test_many_tokens(b, l, hq, hk, d, rot, dtype, pad, halves):
    """Calls large enough that a warp keeps several heads' rows under way (from
    148 * 48 warps on) and, in the gradient, takes several chunks (from 888
    blocks of four warps on): at most 6 chunks of 8 rows a lane, so dw's longest
    chain is 48 + 2 (lane groups) + 4 (warps) + 28 + 32 (blocks) additions."""
    g = _gen(l + d)
    qkv = (torch.randn(b, l, hq + 2 * hk, d + pad, device="cuda", generator=g)
           * torch.exp(torch.randn(b, l, 1, 1, device="cuda", generator=g))).to(dtype)[..., pad:]
    q, k = qkv[:, :, :hq], qkv[:, :, hq + hk:]
    wq, wk = (torch.randn(d, device="cuda", generator=g).to(dtype) for _ in range(2))
    rope = _table(l, rot // 2, g, b)
    how = {"norm_q_w": wq, "norm_k_w": wk, "rope": rope, "rope_halves": halves}
    yq, yk = qk_norm_rope(q, k, **how)
    _check_forward(yq, q, wq, rope, halves, 1e-6, True)
    _check_forward(yk, k, wk, rope, halves, 1e-6, True)
    dq, dk = (torch.randn(b, l, h, d + pad, device="cuda", generator=g).to(dtype)[..., pad:] for h in (hq, hk))
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, **how)
    _check_backward(gq, gwq, dq, q, wq, rope, halves, 1e-6, True)
    _check_backward(gk, gwk, dk, k, wk, rope, halves, 1e-6, True)
    again = qk_norm_rope_backward(dq, dk, q, k, **how)
    assert all(torch.equal(x, y) for x, y in zip((gq, gk, gwq, gwk), again))


def test_upstream_gradients_of_a_sum_and_of_a_transposed_use():
    g = _gen(18)
    q = torch.randn(2, 9, 5, 64, device="cuda", generator=g).bfloat16()
    k = torch.randn(2, 9, 2, 64, device="cuda", generator=g).bfloat16()
    w = torch.randn(64, device="cuda", generator=g)
    rope = _table(9, 32, g)
    dq = torch.ones((), device="cuda", dtype=BF16).expand(q.shape)
    dk = torch.randn(64, 2, 9, 2, device="cuda", generator=g).bfloat16().permute(1, 2, 3, 0)
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, norm_q_w=w, norm_k_w=w, rope=rope)
    _check_backward(gq, gwq, dq, q, w, rope, False, 1e-6, True)
    _check_backward(gk, gwk, dk, k, w, rope, False, 1e-6, True)


@pytest.mark.parametrize("halves", [False, True])
def test_in_place_is_the_same(halves):
    g = _gen(4)
    qkv = torch.randn(2, 70, 24, 128, device="cuda", generator=g).bfloat16()
    rope = _table(70, 48, g)
    w = torch.randn(128, device="cuda", generator=g).bfloat16()
    q, k, v = qkv[:, :, :16], qkv[:, :, 16:20], qkv[:, :, 20:].clone()
    want = qk_norm_rope(q, k, norm_q_w=w, norm_k_w=w, rope=rope, rope_halves=halves)
    got = qk_norm_rope(q, k, norm_q_w=w, norm_k_w=w, rope=rope, rope_halves=halves, q_out=q, k_out=k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(qkv[:, :, 20:], v)


def test_q_alone_expanded_and_empty():
    g = _gen(5)
    q = torch.randn(1, 13, 1, 128, device="cuda", generator=g).half().expand(3, 13, 6, 128)
    w = torch.randn(128, device="cuda", generator=g).half()
    y, none = qk_norm_rope(q, norm_q_w=w)
    assert none is None
    _check_forward(y, q, w, None, False, 1e-6, True)
    gq, gk, gwq, gwk = qk_norm_rope_backward(torch.ones_like(y), None, q, norm_q_w=w)
    assert gq.shape == q.shape and gk is None and gwk is None
    _check_backward(gq, gwq, torch.ones_like(y), q, w, None, False, 1e-6, True)
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64), (2, 5, 0, 64)):
        e = torch.empty(shape, device="cuda", dtype=BF16)
        ones = torch.ones(64, device="cuda", dtype=BF16)
        y, _ = qk_norm_rope(e, norm_q_w=ones)
        assert y.shape == shape
        gq, _, gw, _ = qk_norm_rope_backward(e, None, e, norm_q_w=ones)
        assert gq.shape == shape and (gw == 0).all()


def test_zero_rows_infinities_and_nan_stay_in_their_row():
    g = _gen(6)
    x = torch.randn(1, 6, 4, 128, device="cuda", generator=g).bfloat16()
    clean = x.clone()
    x[0, 1, 2] = 0
    x[0, 3, 1, 5] = float("nan")
    x[0, 4, 0, 7] = float("inf")
    rope = _table(6, 32, g)
    y, _ = qk_norm_rope(x, rope=rope)
    want, _ = qk_norm_rope(clean, rope=rope)
    assert (y[0, 1, 2] == 0).all()
    assert y[0, 3, 1].isnan().all()
    assert y[0, 4, 0, 7].isnan()
    mask = torch.ones(6, 4, dtype=torch.bool, device="cuda")
    mask[1, 2] = mask[3, 1] = mask[4, 0] = False
    assert torch.equal(y[0][mask], want[0][mask])
    # rotation alone: an infinity reaches its partner and no value past the rotated ones
    x = clean.clone()
    x[0, 0, 0, 100] = float("inf")
    y, _ = qk_norm_rope(x, norm_mode=_lib.NORM_NONE, rope=rope)
    assert torch.equal(y[0, 0, 0, 64:], x[0, 0, 0, 64:])


@pytest.mark.parametrize("d", [64, 128])
def test_no_eps(d):
    """Heads that do not fill a warp's lane groups, without an eps."""
    g = _gen(17)
    q, dq = (torch.randn(2, 5, 3, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    k, dk = (torch.randn(2, 5, 1, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    wq, wk = (torch.randn(d, device="cuda", generator=g) for _ in range(2))
    rope = _table(5, d // 2, g)
    how = {"norm_q_w": wq, "norm_k_w": wk, "eps": 0.0, "rope": rope}
    yq, yk = qk_norm_rope(q, k, **how)
    _check_forward(yq, q, wq, rope, False, 0.0, True)
    _check_forward(yk, k, wk, rope, False, 0.0, True)
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, **how)
    _check_backward(gq, gwq, dq, q, wq, rope, False, 0.0, True)
    _check_backward(gk, gwk, dk, k, wk, rope, False, 0.0, True)


def test_gradient_against_differences():
    """fp32 central differences of a 64-bit functional of the kernel's forward."""
    g = _gen(7)
    b, l, h, d = 1, 3, 2, 16
    q = torch.randn(b, l, h, d, device="cuda", generator=g)
    w = torch.randn(d, device="cuda", generator=g)
    rope = _table(l, d // 2, g)
    up = torch.randn(b, l, h, d, device="cuda", generator=g)
    gq, _, gw, _ = qk_norm_rope_backward(up, None, q, norm_q_w=w, rope=rope)

    def value(q, w):
        return float((qk_norm_rope(q, norm_q_w=w, rope=rope)[0].double() * up.double()).sum())

    # h^2 / 6 times a third derivative (here below 1e3) and 2^-20 * sum |terms| / h: h = 2^-7 keeps both below 3e-2
    step = 2.0 ** -7
    for t, grad in ((q, gq), (w, gw)):
        for at in (0, t.numel() // 2, t.numel() - 1):
            hi, lo = t.flatten().clone(), t.flatten().clone()
            hi[at] += step
            lo[at] -= step
            args = [(hi.view(t.shape), w), (lo.view(t.shape), w)] if t is q else [(q, hi), (q, lo)]
            slope = (value(*args[0]) - value(*args[1])) / float(hi[at] - lo[at])
            assert abs(slope - float(grad.flatten()[at])) < 3e-2 * max(1.0, abs(slope))


def test_streams_graphs_and_two_calls_at_once():
    g = _gen(8)
    q = torch.randn(2, 300, 8, 128, device="cuda", generator=g).bfloat16()
    k = torch.randn(2, 300, 2, 128, device="cuda", generator=g).bfloat16()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    w = torch.randn(128, device="cuda", generator=g).bfloat16()
    rope = _table(300, 64, g)
    how = {"norm_q_w": w, "norm_k_w": w, "rope": rope}
    want = (*qk_norm_rope(q, k, **how), *qk_norm_rope_backward(dq, dk, q, k, **how))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([(*qk_norm_rope(q, k, **how), *qk_norm_rope_backward(dq, dk, q, k, **how)) for _ in range(4)])
    torch.cuda.synchronize()
    for per in got:
        for outs in per:
            assert all(torch.equal(x, y) for x, y in zip(outs, want))
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed in turn on new data
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = (*qk_norm_rope(q, k, **how), *qk_norm_rope_backward(dq, dk, q, k, **how))
        graphs.append((graph, outs))
    q.copy_(torch.randn_like(q))
    want = (*qk_norm_rope(q, k, **how), *qk_norm_rope_backward(dq, dk, q, k, **how))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_one_plan_on_another_alignment_and_from_two_threads():
    """Sizes and strides alike, bases on 16 bytes and 2 past them; and two threads that call at the same time."""
    import threading

    g = _gen(19)
    w = torch.randn(64, device="cuda", generator=g).bfloat16()
    rope = _table(50, 32, g)
    how = {"norm_q_w": w, "norm_k_w": w, "rope": rope}
    flat = torch.randn(2 * 50 * 6 * 64 + 8, device="cuda", generator=g).bfloat16()
    up = torch.randn(2 * 50 * 6 * 64 + 8, device="cuda", generator=g).bfloat16()

    def at(t, first):
        return t[first:first + 2 * 50 * 6 * 64].view(2, 50, 6, 64)

    def call(first):
        q, dq = at(flat, first), at(up, first)
        return (*qk_norm_rope(q[:, :, :4], q[:, :, 4:], **how),
                *qk_norm_rope_backward(dq[:, :, :4], dq[:, :, 4:], q[:, :, :4], q[:, :, 4:], **how))

    want = {}
    for first in (0, 1, 8, 3):
        yq, yk, gq, gk, gwq, gwk = want[first] = call(first)
        q, dq = at(flat, first), at(up, first)
        _check_forward(yq, q[:, :, :4], w, rope, False, 1e-6, True)
        _check_forward(yk, q[:, :, 4:], w, rope, False, 1e-6, True)
        _check_backward(gq, gwq, dq[:, :, :4], q[:, :, :4], w, rope, False, 1e-6, True)
        _check_backward(gk, gwk, dq[:, :, 4:], q[:, :, 4:], w, rope, False, 1e-6, True)
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(first):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                got[first] = [call(first) for _ in range(50)]
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 - shown below, from the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(first,)) for first in want]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for first, calls in got.items():
        assert all(torch.equal(x, y) for outs in calls for x, y in zip(outs, want[first]))


def test_matches_the_fused_prologue_up_to_its_roundings():
    """prologue.qkv_prologue_scatter at world 1 rounds to bf16 after the norm
    and after the weight as well: three roundings of 2^-8 (the first two of
    terms of the rotation) against one here."""
    from dgx_monarch_b200.prologue import qkv_prologue_scatter, rope_table

    g = _gen(9)
    q, k, v = (torch.randn(1, 40, 4, 128, device="cuda", generator=g).bfloat16() for _ in range(3))
    w = (1 + 0.1 * torch.randn(128, device="cuda", generator=g)).bfloat16()
    pos = torch.stack([torch.arange(40, device="cuda"), torch.arange(40, device="cuda") % 7], 1)
    rope = rope_table(pos, [64, 64])
    recv = [torch.zeros(1, 40, 4, 128, device="cuda", dtype=BF16) for _ in range(3)]
    qkv_prologue_scatter(q, k, v, [[r.data_ptr()] for r in recv], world=1, rank=0, norm_mode=_lib.NORM_HEAD,
                         norm_q_w=w, norm_k_w=w, rope=rope)
    got = qk_norm_rope(q, k, norm_q_w=w, norm_k_w=w, rope=rope)
    for a, r, x in zip(got, recv, (q, k)):
        v64 = x.double()
        n = v64 / (v64.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        _, size = _turn(n, rope, False)
        assert ((a.double() - r.double()).abs() <= 2.0 ** -8 * 4.1 * size).all()

"""The block norm and its gradient on the GPU against 64 bits (block_reference
derives the limits)."""
from __future__ import annotations

import pytest
import torch

from tests import block_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _mode(name):
    from dgx_monarch_b200 import block_norm as bn

    return {"layer": bn.NORM_LAYER, "rms": bn.NORM_RMS, "none": bn.NORM_NONE}[name]


def make(seed, b, l, c, dtype, *, mode="layer", branch=True, gate="sample", post=False, weights=True, mod="sample",
         mod_dtype=None, weight_dtype=None):
    """Arguments of a call: a stream with uneven rows and channels that stand out."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    shapes = {"shared": (c,), "sample": (b, c), "sample3": (b, 1, c), "token": (b, l, c)}
    md, wd = mod_dtype or dtype, weight_dtype or dtype
    x = rand(b, l, c) * torch.exp(0.5 * rand(b, l, 1)) + 3 * (rand(c) > 2) + 0.2
    a = {"x": x.to(dtype), "branch": rand(b, l, c).to(dtype) if branch else None,
         "gate": rand(*shapes[gate]).to(md) if branch and gate else None, "branch_norm": post,
         "branch_w": (1 + 0.3 * rand(c)).to(wd) if post and weights else None,
         "norm_w": (1 + 0.3 * rand(c)).to(wd) if weights and mode != "none" else None,
         "norm_b": rand(c).to(wd) if weights and mode == "layer" else None,
         "scale": (0.5 * rand(*shapes[mod])).to(md) if mod and mode != "none" else None,
         "shift": rand(*shapes[mod]).to(md) if mod and mode != "none" else None}
    up = {"dy": None if mode == "none" else rand(b, l, c).to(dtype), "dr": rand(b, l, c).to(dtype)}
    return a, up


def run_forward(a, mode, **kw):
    from dgx_monarch_b200.block_norm import block_norm

    r, y = block_norm(**a, norm_mode=_mode(mode), **kw)
    want_r, want_y, r_err, y_err = ref.forward(**a, mode=mode)
    if a["branch"] is not None:
        ref.check("x_out", r, want_r, r_err)
    if mode != "none":
        ref.check("out", y, want_y, y_err)
    return r, y


def run_backward(a, up, mode, r=None):
    from dgx_monarch_b200.block_norm import block_norm_backward

    a = dict(a)
    x = a.pop("x") if r is None else r
    a.pop("x", None)
    grads = block_norm_backward(up["dy"], up["dr"], x, norm_mode=_mode(mode), **a)
    want = ref.backward(up["dy"], up["dr"], x, mode=mode, **a)
    for name, value in grads._asdict().items():
        assert (value is None) == (a.get(name) is None if name != "x" else False), name
        if value is not None:
            ref.check(name, value, *want[name])
            assert value.dtype == (x if name == "x" else a[name]).dtype
    return grads


@pytest.mark.parametrize("width", [1, 3, 8, 24, 31, 64, 257, 512, 1000, 1365, 1536, 2730, 4096, 5120, 5121, 8192])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
def test_widths(width, kind):
    a, up = make(width, 2, 5, width, TYPES[kind])
    run_forward(a, "layer")
    run_backward(a, up, "layer")


@pytest.mark.parametrize("mode", ["layer", "rms", "none"])
@pytest.mark.parametrize("gate,mod", [("shared", "shared"), ("sample", "sample"), ("sample3", "sample3"), ("token", "token"),
                                      ("token", "sample"), ("sample", "token"), (None, None), ("shared", "token")])
@pytest.mark.parametrize("post", [False, True])
def test_forms(mode, gate, mod, post):
    for width in (640, 333):
        a, up = make(7, 3, 11, width, torch.bfloat16, mode=mode, gate=gate, mod=mod, post=post)
        run_forward(a, mode)
        run_backward(a, up, mode)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("gate,mod", [("sample", "sample"), ("token", "token")])
def test_modulation_and_weights_of_fp32(kind, gate, mod):
    for width in (520, 777):
        a, up = make(3, 2, 9, width, TYPES[kind], gate=gate, mod=mod, post=True, mod_dtype=torch.float32,
                     weight_dtype=torch.float32)
        run_forward(a, "layer")
        run_backward(a, up, "layer")


@pytest.mark.parametrize("drop", ["branch", "gate", "weights", "scale", "shift", "dr", "all"])
@pytest.mark.parametrize("mode", ["layer", "rms"])
def test_absent_arguments(drop, mode):
    a, up = make(11, 2, 6, 320, torch.float16, mode=mode, post=drop == "gate")
    gone = {"branch": ["branch", "gate"], "weights": ["norm_w", "norm_b"], "dr": [],
            "all": ["branch", "gate", "norm_w", "norm_b", "scale", "shift"]}.get(drop, [drop])
    a.update({n: None for n in gone})
    if drop in ("dr", "all"):
        up["dr"] = None
    run_forward(a, mode)
    run_backward(a, up, mode)


@pytest.mark.parametrize("b,l", [(1, 1), (1, 2), (3, 1), (1, 148), (2, 1023), (70, 3), (1, 5000)])
@pytest.mark.parametrize("width", [192, 1283])
def test_row_counts(b, l, width):
    """From one row to several a block, samples that end inside a block's rows, more samples than warps of the last sum."""
    a, up = make(b + l, b, l, width, torch.bfloat16, post=l % 2 == 1)
    run_forward(a, "layer")
    run_backward(a, up, "layer")


@pytest.mark.parametrize("gate,mod", [("sample", "sample"), ("sample3", "token"), ("shared", "sample3"), ("token", "shared"), (None, "sample")])
@pytest.mark.parametrize("b,width", [(2, 192), (3, 1283), (700, 520)])
def test_samples_of_one_row(b, width, gate, mod):
    """Values of a sample that has one row; also slices of a wider projection, samples far apart."""
    a, up = make(b, b, 1, width, torch.bfloat16, gate=gate, mod=mod, post=b == 3)
    run_forward(a, "layer")
    run_backward(a, up, "layer")
    for name in ("x", "branch", "gate", "scale", "shift"):
        t = a[name]
        if t is not None and t.ndim > 1:
            wide = torch.zeros(*t.shape[:-1], 2 * width + 8, device="cuda", dtype=t.dtype)
            a[name] = wide[..., 8:8 + width].copy_(t)
    run_forward(a, "rms" if a["norm_b"] is None else "layer")
    run_backward(a, up, "layer")


@pytest.mark.parametrize("b,l", [(0, 4), (2, 0)])
def test_no_rows(b, l):
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    a, up = make(0, b, l, 64, torch.bfloat16)
    r, y = block_norm(**a, norm_mode=_mode("layer"))
    assert r.shape == y.shape == (b, l, 64)
    x = a.pop("x")
    grads = block_norm_backward(up["dy"], up["dr"], x, norm_mode=_mode("layer"), **a)
    for name in ("gate", "scale", "shift", "norm_w", "norm_b"):
        assert torch.equal(getattr(grads, name), torch.zeros_like(a[name])), name


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strides(offset):
    """Slices of wider tensors (rows on and off 16 bytes), batch and rows exchanged, expanded inputs, chunks of a projection."""
    from dgx_monarch_b200.block_norm import block_norm

    b, l, c = 2, 6, 200
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(b, l, 3 * c + 24, device="cuda", generator=g).bfloat16()
    x = wide[..., offset:offset + c]
    branch = torch.randn(l, b, c, device="cuda", generator=g).bfloat16().transpose(0, 1)
    six = torch.randn(b, 6 * c + 1, device="cuda", generator=g).bfloat16()
    parts = [six[:, offset + i * c:offset + (i + 1) * c] for i in range(3)]
    a = {"x": x, "branch": branch, "gate": parts[0], "scale": parts[1], "shift": parts[2]}
    run_forward(a, "layer")
    dy = torch.randn(b, l, 2 * c, device="cuda", generator=g).bfloat16()
    for up in ({"dy": dy[..., offset:offset + c], "dr": dy[..., c - offset:2 * c - offset]},
               {"dy": dy[..., ::2], "dr": torch.ones((), device="cuda", dtype=x.dtype).expand(b, l, c)}):
        run_backward(a, up, "layer")
    run_forward({**a, "x": x[:1, :1].expand(b, l, c)}, "rms")
    # outputs that are slices: what lies beside them stays
    room = torch.full((2, b, l, c + 16), 7.0, device="cuda", dtype=x.dtype)
    r, y = room[0, ..., offset:offset + c], room[1, ..., offset:offset + c]
    got_r, got_y = block_norm(**a, x_out=r, out=y)
    assert got_r is r and got_y is y
    want_r, want_y = block_norm(**a)
    assert torch.equal(r, want_r) and torch.equal(y, want_y)
    assert (room[..., :offset] == 7).all() and (room[..., offset + c:] == 7).all()


@pytest.mark.parametrize("width", [512, 515])
def test_in_place(width):
    from dgx_monarch_b200.block_norm import block_norm

    a, _ = make(2, 2, 40, width, torch.bfloat16, post=True)
    want_r, want_y = block_norm(**a)
    for r_of, y_of in (("x", "branch"), ("branch", "x"), ("x", None), (None, "branch")):
        c = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in a.items()}
        r, y = block_norm(**c, x_out=c[r_of] if r_of else None, out=c[y_of] if y_of else None)
        assert torch.equal(r, want_r) and torch.equal(y, want_y)


@pytest.mark.parametrize("mode", ["layer", "rms"])
@pytest.mark.parametrize("width", [640, 643])
def test_rows_that_are_not_finite_stay_alone(mode, width):
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    a, up = make(4, 1, 50, width, torch.bfloat16, mode=mode, gate="token", mod="token")
    want_r, want_y = block_norm(**a, norm_mode=_mode(mode))
    bad = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in a.items()}
    bad["x"][0, 7, 5] = float("nan")
    bad["x"][0, 20, width - 1] = float("inf")
    bad["branch"][0, 33, 0] = float("-inf")
    r, y = block_norm(**bad, norm_mode=_mode(mode))
    fine = torch.ones(50, dtype=torch.bool, device="cuda")
    fine[[7, 20, 33]] = False
    assert torch.equal(y[0, fine], want_y[0, fine]) and torch.equal(r[0, fine], want_r[0, fine])
    assert y[0, 7].isnan().all() and y[0, 20, width - 1].isnan() and y[0, 33, 0].isnan()
    rest = {n: t for n, t in a.items() if n != "x"}
    good = block_norm_backward(up["dy"], up["dr"], a["x"], norm_mode=_mode(mode), **rest)
    rest["branch"] = bad["branch"]
    got = block_norm_backward(up["dy"], up["dr"], bad["x"], norm_mode=_mode(mode), **rest)
    for name in ("x", "branch", "gate", "scale", "shift"):
        assert torch.equal(getattr(got, name)[0, fine], getattr(good, name)[0, fine]), name


def test_values_at_the_ends_of_the_range():
    """A constant row (no deviation), zeros, and rows far from zero beside their spread."""
    c = 1024
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, 6, c, device="cuda", generator=g)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = 5.0, 0.0, x[0, 2] * 1e-12, x[0, 3] * 1e15
    x[0, 4] += 1000
    a = {"x": x, "branch": None}
    for mode in ("layer", "rms"):
        run_forward(a, mode)
        run_backward(a, {"dy": torch.randn(1, 6, c, device="cuda", generator=g), "dr": None}, mode)


def test_gradient_against_differences_of_the_kernel():
    """fp32: central differences of step h over both outputs; rounding of the forward leaves about
    2^-24 sqrt(values) / h of the loss' size, the third derivative h^2."""
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    a, up = make(9, 2, 33, 384, torch.float32, mode="layer", gate="sample", mod="sample", post=True)
    up = {n: t.double() for n, t in up.items()}

    def loss(args):
        r, y = block_norm(**args)
        return (r.double() * up["dr"]).sum() + (y.double() * up["dy"]).sum()

    r, _ = block_norm(**a)
    rest = {n: t for n, t in a.items() if n != "x"}
    grads = block_norm_backward(up["dy"].float(), up["dr"].float(), r, **rest)
    h = 2.0 ** -8
    for name, value in a.items():
        if not isinstance(value, torch.Tensor):
            continue
        way = torch.sign(torch.randn(value.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)))
        plus, minus = value + h * way, value - h * way
        diff = (loss({**a, name: plus}) - loss({**a, name: minus})) / (2 * h)
        grad = getattr(grads, name).double()
        want = (grad * (plus - minus).double() / (2 * h)).sum()
        # The loss is a sum of 2 * 2 * 33 * 384 products of size about 1 with independent roundings of 2^-22 each (four
        # operations): 2^-22 * sqrt(50688) / h = 0.014; the step's own error is h^2 / 6 of third derivatives of order one
        # in random directions: 1e-5 * sqrt(50688) = 0.0006.  Six times their sum.
        assert abs(diff - want) <= 0.09, (name, diff, want)


def test_same_bits_streams_and_graphs():
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    a, up = make(5, 2, 700, 1536, torch.bfloat16, post=True)
    rest = {n: t for n, t in a.items() if n != "x"}
    first = block_norm(**a)
    grads = block_norm_backward(up["dy"], up["dr"], a["x"], **rest)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block_norm(**a)
        others = block_norm_backward(up["dy"], up["dr"], a["x"], **rest)
    side.synchronize()
    for x, y in zip(first + tuple(grads), other + tuple(others)):
        assert torch.equal(x, y)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(block_norm(**a) + tuple(block_norm_backward(up["dy"], up["dr"], a["x"], **rest)))
        graphs.append(graph)
    a["x"].copy_(a["x"].flip(1))
    up["dy"].neg_()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = block_norm(**a) + tuple(block_norm_backward(up["dy"], up["dr"], a["x"], **rest))
    for out in outs:
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_many_calls_in_a_row():
    """Rows that land out of order must not be taken for those before them in the ring: the wait would run out (and set the
    device error), or a row come out wrong."""
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    for width, rows in ((5120, 4000), (2048, 6000), (8192, 2000), (1365, 4000)):
        a, up = make(8, 1, rows, width, torch.bfloat16)
        rest = {n: t for n, t in a.items() if n != "x"}
        want, grads = block_norm(**a), block_norm_backward(up["dy"], up["dr"], a["x"], **rest)
        for _ in range(60):
            got = block_norm(**a)
            more = block_norm_backward(up["dy"], up["dr"], a["x"], **rest)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(more, grads) if x is not None)

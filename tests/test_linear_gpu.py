"""The 16-bit Linear and its gradients on the GPU against 64 bits.

Limits: a sum over K products in fp32 passes K / 16 accumulations of the
tensor core and the alignment of each sixteen products, 2^-23 of the sum of
magnitudes each: (K / 8 + 16) 2^-23 covers both.  exp, its quotient and erf
leave an activation off by less than 2^-20 of |z| and its slope by less than
2^-19 (1 + |z|).
"""
from __future__ import annotations

import math

import pytest
import torch

from tests.block_reference import U, check, half_step, lift, tiny

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ["none", "silu", "gelu", "gelu_tanh"]


def act(z, name):
    f = torch.nn.functional
    return {"none": lambda v: v, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[name](z)


def slope(z, name):
    with torch.enable_grad():
        v = z.detach().clone().requires_grad_(True)
        return torch.autograd.grad(act(v, name).sum(), v)[0]


def make(seed, lead, n, k, dtype, *, gate=None, bias=True, residual=False, gate_dtype=None, out_dtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    shapes = {"shared": (n,), "sample": (lead[0], n), "sample3": (lead[0], 1, n), "token": (*lead, n)}
    a = {"x": (rand(*lead, k) + 0.2).to(dtype), "w": (rand(n, k) * k ** -0.5).to(dtype),
         "bias": rand(n).to(dtype) if bias else None, "gate": rand(*shapes[gate]).to(gate_dtype or dtype) if gate else None}
    res = rand(*lead, n).to(out_dtype or dtype) if residual else None
    return a, res, rand(*lead, n).to(dtype)


def gate_of(a):
    gate = a["gate"]
    if gate is None:
        return torch.ones((), dtype=torch.float64, device="cuda")
    if a["x"].ndim == 2:
        return gate.double()
    return lift(gate, a["x"].shape[1])


def run_forward(a, res, name="none", **kw):
    from dgx_monarch_b200.linear import linear

    got, pre = linear(**a, activation=name, residual=res, return_pre=True, **kw)
    x, w = a["x"].double(), a["w"].double()
    k = x.shape[-1]
    z = x @ w.T
    z_err = (k / 8 + 16) * 2 * U * (x.abs() @ w.abs().T)
    if a["bias"] is not None:
        z = z + a["bias"].double()
    z_err = z_err + 2 * U * z.abs()
    check("pre", pre, z, z_err)
    g = gate_of(a)
    want = act(z, name) * g
    err = g.abs() * (1.13 * z_err + (0 if name == "none" else 2.0 ** -20 * z.abs())) + 4 * U * want.abs()
    if res is not None:
        want = want + res.double()
        err = err + 2 * U * (res.double().abs() + want.abs())
    check("out", got, want, err)
    return got, pre


def run_backward(a, dout, name="none", pre=None, **kw):
    from dgx_monarch_b200.linear import linear_backward

    if pre is None and (name != "none" or a["gate"] is not None):
        pre = (a["x"].float() @ a["w"].float().T).to(a["x"].dtype)
    grads = linear_backward(dout, a["x"], a["w"], bias=a["bias"], activation=name, gate=a["gate"], pre=pre, **kw)
    dtype, half = a["x"].dtype, half_step(a["x"].dtype)
    x, w, up, g = a["x"].double().flatten(0, -2), a["w"].double(), dout.double(), gate_of(a)
    z = torch.zeros_like(up) if pre is None else pre.double()
    dz = up * g * slope(z, name)
    dz_err = 4 * U * dz.abs() + (0 if name == "none" else 2.0 ** -19 * (1 + z.abs()) * (up * g).abs())
    m, n = dz.shape[:-1].numel(), dz.shape[-1]
    exact_dz = name == "none" and a["gate"] is None and dout.dtype == dtype
    rounded = 0 * dz_err if exact_dz else half * dz.abs() + (1 + half) * dz_err + tiny(dtype)
    flat, flat_err, size = dz.flatten(0, -2), rounded.flatten(0, -2), dz.abs().flatten(0, -2)
    if grads.x is not None:
        err = flat_err @ w.abs() + (n / 8 + 16) * 2 * U * ((size + flat_err) @ w.abs())
        check("x", grads.x, (flat @ w).view(a["x"].shape), err.view(a["x"].shape))
    if grads.w is not None:
        err = flat_err.T @ x.abs() + (m / 8 + 16) * 2 * U * ((size + flat_err).T @ x.abs())
        check("w", grads.w, flat.T @ x, err)
    if a["bias"] is not None:
        check("bias", grads.bias, flat.sum(0), dz_err.flatten(0, -2).sum(0) + (m + 64) * U * size.sum(0))
    if a["gate"] is not None:
        value = up * act(z, name)
        err = up.abs() * (2.0 ** -20 * z.abs() + 2 * U * act(z, name).abs())
        gate = a["gate"]
        if gate.ndim == 1:
            value, err, mag = value.flatten(0, -2).sum(0), err.flatten(0, -2).sum(0), value.abs().flatten(0, -2).sum(0)
        elif gate.shape != value.shape:
            value, err, mag = value.sum(1).view(gate.shape), err.sum(1).view(gate.shape), value.abs().sum(1).view(gate.shape)
        else:
            mag = 0 * value
        check("gate", grads.gate, value, err + (m + 64) * U * mag)
    return grads


SIZES = [(1, 8, 16), (1, 1, 1), (1, 5120, 512), (2, 300, 100), (7, 129, 65), (16, 256, 64), (17, 1000, 192), (33, 64, 1003),
         (64, 512, 2048), (65, 128, 128), (100, 1, 9), (128, 777, 320), (200, 130, 3), (257, 256, 256), (300, 1000, 72),
         (511, 2048, 128), (1024, 1024, 512), (2050, 1030, 200), (3000, 513, 65), (1, 30000, 64)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_sizes(m, n, k, kind):
    """Every tile, split and order of operands; sizes that fill no tile, word or stage."""
    a, res, dout = make(m + n + k, (m,), n, k, TYPES[kind], residual=m % 2 == 0)
    run_forward(a, res)
    run_backward(a, dout)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("gate", [None, "shared", "sample", "sample3", "token"])
@pytest.mark.parametrize("lead,n,k", [((3, 5), 72, 40), ((2, 150), 264, 136), ((2, 300), 515, 77), ((1, 1), 512, 256)])
def test_epilogues(name, gate, lead, n, k):
    a, res, dout = make(7, lead, n, k, torch.bfloat16, gate=gate, residual=True)
    _, pre = run_forward(a, res, name)
    run_backward(a, dout, name, pre)


@pytest.mark.parametrize("m", [2, 40, 700])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_fp32_outputs_bias_gate_and_gradients(m, kind):
    dtype = TYPES[kind]
    a, res, dout = make(5, (2, m), 200, 96, dtype, gate="sample", residual=True, gate_dtype=torch.float32,
                        out_dtype=torch.float32)
    a["bias"] = a["bias"].float()
    got, pre = run_forward(a, res, "gelu", out_dtype=torch.float32)
    assert got.dtype == torch.float32 and pre.dtype == dtype
    grads = run_backward(a, dout.float(), "gelu", pre)
    assert grads.bias.dtype == grads.gate.dtype == torch.float32
    run_backward({**a, "gate": None}, dout.float())


def test_long_k():
    """A sum over more stages than the ring holds many times over, alone and split."""
    for m in (1, 300):
        a, res, dout = make(3, (m,), 136, 20000, torch.bfloat16)
        run_forward(a, res)
    a, res, dout = make(3, (9000,), 136, 64, torch.bfloat16)
    run_backward(a, dout)


@pytest.mark.parametrize("m,n,k", [(200, 136, 4096), (257, 72, 2051), (70, 400, 1600), (1000, 8, 1024), (65, 129, 515)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_few_tiles(m, n, k, dtype):
    """Products whose K is shared among CTAs, in each direction, with several tiles of rows and everything in the epilogue."""
    a, res, dout = make(m, (m,), n, k, dtype, gate="token", residual=True)
    _, pre = run_forward(a, res, "silu")
    run_backward(a, dout, "silu", pre)
    a, res, dout = make(m, (m,), n, k, dtype, gate="shared")
    run_forward(a, res, out_dtype=torch.float32)
    a, res, dout = make(m, (k,), n, m, dtype)  # w's gradient along k rows
    run_backward(a, dout)


@pytest.mark.parametrize("samples", [1, 2, 3, 31, 33, 70])
def test_sums_over_samples(samples):
    a, res, dout = make(samples, (samples, 9), 40, 64, torch.bfloat16, gate="sample")
    run_backward(a, dout, "gelu")
    a["gate"] = a["gate"][0].clone()
    run_backward(a, dout, "gelu")


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strides(offset):
    """Slices (on and off 16 bytes), batch and rows exchanged, a transposed weight, expanded tensors, outputs beside others."""
    from dgx_monarch_b200.linear import linear

    b, l, n, k = 2, 70, 200, 96
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    room = rand(b, l, 3 * k)
    x = room[..., offset:offset + k]
    a = {"x": x, "w": rand(n, 2 * k)[:, offset:offset + k], "bias": rand(n), "gate": rand(b, 6 * n)[:, offset:offset + n]}
    res = rand(b, l, n + 24)[..., offset:offset + n]
    _, pre = run_forward(a, res, "silu")
    run_backward(a, rand(b, l, 2 * n)[..., offset:offset + n], "silu", pre)
    run_backward(a, torch.ones((), device="cuda", dtype=x.dtype).expand(b, l, n), "silu", pre)
    a2 = {"x": rand(l, b, k).transpose(0, 1), "w": rand(k, n).T, "bias": None, "gate": None}
    run_forward(a2, rand(1, 1, n).expand(b, l, n))
    run_backward(a2, rand(l, b, n).transpose(0, 1))
    run_forward({**a2, "x": rand(1, 1, k).expand(b, l, k)}, None)
    wide = torch.full((b, l, n + 32), 7.0, device="cuda", dtype=x.dtype)
    out = wide[..., offset:offset + n]
    got = linear(**a, residual=res, out=out)
    assert got is out and torch.equal(out, linear(**a, residual=res))
    assert (wide[..., :offset] == 7).all() and (wide[..., offset + n:] == 7).all()


@pytest.mark.parametrize("m,n", [(3, 256), (130, 256), (1100, 1024), (130, 259)])
def test_output_on_its_residual(m, n):
    from dgx_monarch_b200.linear import linear

    a, res, _ = make(8, (1, m), n, 128, torch.bfloat16, gate="shared", residual=True)
    want = linear(**a, residual=res)
    stream = res.clone()
    assert linear(**a, residual=stream, out=stream) is stream
    assert torch.equal(stream, want)


def test_empty():
    from dgx_monarch_b200.linear import linear, linear_backward

    a, _, dout = make(0, (2, 0), 16, 32, torch.bfloat16, gate="shared")
    assert linear(**a).shape == (2, 0, 16)
    grads = linear_backward(dout, a["x"], a["w"], bias=a["bias"], gate=a["gate"], pre=dout)
    assert grads.x.shape == (2, 0, 32)
    for got, like in ((grads.w, a["w"]), (grads.bias, a["bias"]), (grads.gate, a["gate"])):
        assert torch.equal(got, torch.zeros_like(like))
    a, _, dout = make(0, (3,), 0, 32, torch.bfloat16, bias=False)
    assert linear(**a).shape == (3, 0)
    assert torch.equal(linear_backward(dout, a["x"], a["w"]).x, torch.zeros_like(a["x"]))


@pytest.mark.parametrize("m,n,k", [(5, 300, 128), (260, 300, 128), (1100, 1024, 192)])
def test_rows_that_are_not_finite_stay_alone(m, n, k):
    from dgx_monarch_b200.linear import linear

    a, res, _ = make(1, (m,), n, k, torch.bfloat16, residual=True)
    want = linear(**a, residual=res, activation="gelu")
    a["x"] = a["x"].clone()
    a["x"][2, 3] = float("nan")
    a["x"][m - 1, 0] = float("inf")
    got = linear(**a, residual=res, activation="gelu")
    fine = torch.ones(m, dtype=torch.bool, device="cuda")
    fine[[2, m - 1]] = False
    assert torch.equal(got[fine], want[fine]) and got[2].isnan().all() and not got[m - 1].isfinite().all()


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_activations_at_the_ends_of_the_range(name):
    from dgx_monarch_b200.linear import linear

    z = torch.tensor([-6e4, -1e4, -100.0, -20.0, -8.0, -1e-3, -0.0, 0.0, 1e-3, 8.0, 20.0, 100.0, 1e4, 6e4], device="cuda")
    a = {"x": torch.ones(3, 8, device="cuda").bfloat16(), "w": torch.zeros(z.numel(), 8, device="cuda").bfloat16(), "bias": z}
    got = linear(**a, activation=name, out_dtype=torch.float32)
    want = act(z.double(), name).expand(3, -1)
    assert ((got.double() - want).abs() <= 2.0 ** -20 * z.double().abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_slopes_at_the_ends_of_the_range(name, dtype):
    """dz of one value a row, x's gradient behind a w of one column of ones: the slope rounded once, 0 or 1 far out."""
    from dgx_monarch_b200.linear import linear_backward

    top = torch.finfo(dtype).max
    z = torch.tensor([[-float("inf"), -top, -1e4, -100.0, -20.0, -8.0, -0.75, -0.0, 0.0, 0.75, 8.0, 20.0, 100.0, 1e4, top,
                       float("inf"), float("nan")]], device="cuda").to(dtype).t().contiguous()
    w = torch.zeros(1, 8, device="cuda", dtype=dtype)
    w[0, 0] = 1
    grads = linear_backward(torch.ones_like(z), torch.zeros(z.shape[0], 8, device="cuda", dtype=dtype), w, activation=name,
                            pre=z, w_grad=False)
    leaf = z.double().clamp(-1e4, 1e4).requires_grad_(True)
    act(leaf, name).sum().backward()
    got, want = grads.x[:, 0].double(), leaf.grad[:, 0]
    assert torch.isnan(got[-1])
    # A rounding; fp32's slope loses 2^-19 of its value where e^-z does (z up to 20), a fp16 of 2^-24 is zero or itself.
    assert ((got - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -18) * want.abs() + 2.0 ** -25)[:-1].all(), (got, want)


def test_gradients_against_differences_of_the_kernel():
    """fp32 outputs, sixteen-bit steps: the Linear is linear in x, w and bias up to the activation; with steps of 2^-4 of
    the 16-bit arguments the third derivative leaves h^2, the sums 2^-20."""
    from dgx_monarch_b200.linear import linear, linear_backward

    g = torch.Generator(device="cuda").manual_seed(4)
    a, _, _ = make(6, (2, 40), 96, 64, torch.float16, gate="sample", gate_dtype=torch.float32)
    a["x"], a["w"] = (torch.round(a["x"].float() * 16) / 16).half(), (torch.round(a["w"].float() * 64) / 64).half()
    a["bias"] = a["bias"].float()
    dout = torch.randn(2, 40, 96, device="cuda", generator=g)
    loss = lambda args: (linear(**args, activation="gelu", out_dtype=torch.float32).double() * dout.double()).sum()
    _, pre = linear(**a, activation="gelu", return_pre=True)
    grads = linear_backward(dout, a["x"], a["w"], bias=a["bias"], activation="gelu", gate=a["gate"], pre=pre)
    for name, h in (("x", 2.0 ** -4), ("w", 2.0 ** -6), ("bias", 2.0 ** -5), ("gate", 2.0 ** -5)):
        way = torch.sign(torch.randn(a[name].shape, device="cuda", generator=g)).to(a[name].dtype)
        diff = (loss({**a, name: a[name] + h * way}) - loss({**a, name: a[name] - h * way})) / (2 * h)
        parts = getattr(grads, name).double() * way.double()
        # Steps along `way` change z by about h |column sums of signs| (0.5 for x and w, 2^-5 for the bias): the third
        # derivative, below 1, leaves (dz)^2 / 6 of the gradient's terms, 4 % each of random sign; 16-bit dz 2^-11.
        limit = 6 * (0.042 + 2.0 ** -10) * parts.flatten().norm() + 1e-3
        assert abs(diff - parts.sum()) <= limit, (name, diff.item(), parts.sum().item(), limit.item())


def test_same_bits_streams_and_graphs():
    from dgx_monarch_b200.linear import linear, linear_backward

    for m, n, k in ((3, 640, 1000), (600, 513, 264), (1500, 1024, 320)):
        a, res, dout = make(5, (1, m), n, k, torch.bfloat16, gate="sample", residual=True)

        def both():
            out, pre = linear(**a, activation="gelu_tanh", residual=res, return_pre=True)
            return (out, pre, *linear_backward(dout, a["x"], a["w"], bias=a["bias"], activation="gelu_tanh", gate=a["gate"],
                                               pre=pre))

        first = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(first, other))
        graphs, outs = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(both())
            graphs.append(graph)
        a["x"].neg_()
        dout.copy_(dout.flip(1))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = both()
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_wanted_gradients_alone():
    from dgx_monarch_b200.linear import linear_backward

    a, _, dout = make(2, (130,), 72, 40, torch.bfloat16)
    whole = linear_backward(dout, a["x"], a["w"], bias=a["bias"])
    for x_grad, w_grad, bias in ((True, False, None), (False, True, None), (False, False, a["bias"])):
        got = linear_backward(dout, a["x"], a["w"], bias=bias, x_grad=x_grad, w_grad=w_grad)
        assert (got.x is None) != x_grad and (got.w is None) != w_grad and (got.bias is None) == (bias is None)
        for one, all_ in zip(got, whole):
            assert one is None or torch.equal(one, all_)
    assert math.isfinite(whole.x.float().sum().item())


@pytest.mark.parametrize("lead,gate", [((2, 0), "shared"), ((2, 0), "sample"), ((2, 0), "sample3"), ((1, 0), "sample"), ((0, 3), "sample"),
                                       ((2, 0), "token"), ((0,), None), ((0,), "one")])
def test_gradients_of_no_rows(lead, gate):
    """Zeros in memory that held something else."""
    from dgx_monarch_b200.linear import linear_backward

    a, _, dout = make(0, lead, 16, 32, torch.bfloat16, gate=None if gate == "one" else gate)
    if gate == "one":
        a["gate"] = torch.ones(1, 16, device="cuda").bfloat16()
    dirty = [torch.full((n,), float("nan"), device="cuda").bfloat16() for n in (16, 32, 16 * 32) for _ in range(4)]
    torch.cuda.synchronize()
    del dirty
    grads = linear_backward(dout, a["x"], a["w"], bias=a["bias"], gate=a["gate"], pre=dout)
    for got, like in ((grads.x, a["x"]), (grads.w, a["w"]), (grads.bias, a["bias"]), (grads.gate, a["gate"])):
        assert (got is None and like is None) or torch.equal(got, torch.zeros_like(like))


@pytest.mark.parametrize("gate", ["shared", "token", "apart", "expanded", "same"])
@pytest.mark.parametrize("b,l", [(1, 1), (700, 1), (1, 700), (233, 3), (5, 131)])
def test_sums_across_samples(b, l, gate):
    """A bias' and a shared gate's sums over many short samples, and tokens' gates: rows a step apart, samples further apart
    than their rows, and one row or one value for all tokens seen as tokens'."""
    a, _, dout = make(b + l, (b, l), 136, 64, torch.bfloat16, gate="shared" if gate == "shared" else "token")
    if gate == "apart":
        wide = torch.zeros(b, l + 2, 136, device="cuda", dtype=torch.bfloat16)
        a["gate"] = wide[:, 1:l + 1].copy_(a["gate"])
    elif gate == "expanded":
        a["gate"] = a["gate"][:, :1].expand(b, l, 136)
    elif gate == "same":
        a["gate"] = a["gate"][:1, :1].expand(b, l, 136)
    for name in ("silu", "none"):
        run_backward(a, dout, name)

"""Linear products of more tiles than the SMs take at one time, so that a CTA or
pair has several: the second accumulator, staging rows that one tile leaves to
the next, and a residual fetched a tile ahead.  Limits as in test_linear_gpu."""
from __future__ import annotations

import pytest
import torch

from tests.block_reference import U, check
from tests.test_linear_gpu import act, gate_of, make, run_backward, run_forward

pytestmark = pytest.mark.gpu

# rows, columns and k that run on single CTAs, and on pairs with tiles of 192 and of 256 columns
SINGLE, PAIR_192, PAIR_256 = (19000, 301, 64), (20000, 515, 64), (20000, 387, 64)


def run(a, res, name="none", **kw):
    """linear without pre against 64 bits."""
    from dgx_monarch_b200.linear import linear

    got = linear(**a, activation=name, residual=res, **kw)
    x, w = a["x"].double(), a["w"].double()
    z = x @ w.T
    z_err = (x.shape[-1] / 8 + 16) * 2 * U * (x.abs() @ w.abs().T)
    if a["bias"] is not None:
        z = z + a["bias"].double()
    z_err = z_err + 2 * U * z.abs()
    g = gate_of(a)
    want = act(z, name) * g
    err = g.abs() * (1.13 * z_err + (0 if name == "none" else 2.0 ** -20 * z.abs())) + 4 * U * want.abs()
    if res is not None:
        want = want + res.double()
        err = err + 2 * U * (res.double().abs() + want.abs())
    check("out", got, want, err)
    return got


@pytest.mark.parametrize("m,n,k", [SINGLE, PAIR_192, PAIR_256])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_residual_on_words_beside_outputs_off_them(m, n, k, out_dtype):
    """The residual comes by bulk loads, the outputs leave by the lanes' stores (rows of n odd values), or by both ways (rows
    on 16 bytes that end inside a word): the loads land where the lanes have just written and read."""
    a, _, _ = make(n, (m,), n, k, torch.bfloat16, gate="shared")
    pitch = (n + 7) // 8 * 8
    res = torch.randn(m, pitch, device="cuda").to(out_dtype)[:, :n]
    apart = run(a, res, out_dtype=out_dtype)
    room = torch.full((m, pitch), 7.0, device="cuda", dtype=out_dtype)
    on_words = run(a, res, out=room[:, :n])
    assert torch.equal(apart, on_words) and (room[:, n:] == 7).all()
    stream = res.clone()
    shared = torch.empty(m, pitch, device="cuda", dtype=out_dtype)[:, :n].copy_(stream)
    from dgx_monarch_b200.linear import linear

    assert torch.equal(linear(**a, residual=shared, out=shared), apart)


# By rows: one tile a CTA or pair at the most, and several.
BY_ROWS = [(300, 1000, 72), (511, 2048, 128), (1100, 1024, 192), SINGLE, PAIR_192, PAIR_256, (19000, 304, 64), (20000, 512, 64),
           (20000, 384, 64)]


@pytest.mark.parametrize("m,n,k", BY_ROWS)
@pytest.mark.parametrize("name", ["none", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=["16", "fp32"])
def test_bias_and_activation_alone(m, n, k, name, out_dtype):
    """The kernels that have nothing else in their epilogue: each activation and output size, on one CTA and on a pair."""
    a, _, _ = make(m + n, (m,), n, k, torch.float16 if n % 3 == 0 else torch.bfloat16)
    run(a, None, name, out_dtype=out_dtype)


@pytest.mark.parametrize("m,n,k", BY_ROWS)
@pytest.mark.parametrize("gate,residual,pre", [("sample", False, False), (None, True, False), ("token", True, True),
                                               ("sample", False, True), ("shared", True, True)])
def test_gate_residual_and_pre(m, n, k, gate, residual, pre):
    """What the rolled epilogue does, over several tiles, with pre by bulk stores, by the lanes and beside a residual."""
    lead = (2, m // 2) if gate == "sample" else (m,)
    a, res, _ = make(m + n, lead, n, k, torch.bfloat16, gate=gate, residual=residual)
    if not pre:
        run(a, res, "silu")
        run(a, None if res is None else res.float(), "gelu", out_dtype=torch.float32)
    else:
        run_forward(a, res, "gelu_tanh")
        run_forward(a, None if res is None else res.float(), "gelu", out_dtype=torch.float32)


@pytest.mark.parametrize("m,n,k", [(19000, 64, 304), (40000, 64, 260), (38000, 64, 128), (20000, 128, 512)])
def test_gradients_of_many_tiles(m, n, k):
    """Products with w's rows contiguous along k, and along the rows, of more tiles than fit at one time."""
    a, _, dout = make(m + k, (m,), n, k, torch.bfloat16)
    run_backward(a, dout, "silu")


@pytest.mark.parametrize("m,n,k", [(70, 4000, 1100), (40, 3001, 2000), (192, 5120, 5128)])
def test_wide_gradients_of_many_tiles(m, n, k):
    """w's gradient of more tiles than CTAs, and than pairs."""
    a, _, dout = make(3, (m,), n, k, torch.bfloat16)
    run_backward(a, dout)

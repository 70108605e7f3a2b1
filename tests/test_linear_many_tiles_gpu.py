"""Linear products of more tiles than the SMs take at one time, so that a CTA or
pair has several: the second accumulator, staging rows that one tile leaves to
the next, and a residual fetched a tile ahead.  Limits as in test_linear_gpu."""
from __future__ import annotations

import pytest
import torch

from tests.block_reference import U, check
from tests.test_linear_gpu import act, gate_of, make

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

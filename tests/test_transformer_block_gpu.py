"""A whole transformer block out of this library's calls, forward and training
step, against 64 bits.

Each call rounds its result once to bf16 (half a step: 2^-8 of a value), as the
block's stages do one after the other, and the stages pass relative errors of
L2 norms on about as they get them: n roundings leave at most n 2^-8.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


def rel(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def _case(seed, b, l, heads, d):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    c, f = heads * d, 3 * heads * d
    lin = lambda n, k: (rand(n, k) * k ** -0.5).bfloat16()
    return {"x": rand(b, l, c).bfloat16(), "mod": 0.3 * rand(b, 6 * c), "qkv": lin(3 * c, c), "qkv_b": (0.1 * rand(3 * c)).bfloat16(),
            "proj": lin(c, c), "up": lin(f, c), "up_b": (0.1 * rand(f)).bfloat16(), "down": lin(c, f),
            "wq": (1 + 0.2 * rand(d)).bfloat16(), "wk": (1 + 0.2 * rand(d)).bfloat16(), "dout": rand(b, l, c).bfloat16()}


def _rope(l, d):
    at = torch.arange(l, device="cuda", dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))
    return torch.stack([at.cos(), at.sin()], dim=-1).float()


def _norm64(x, scale, shift):
    return torch.nn.functional.layer_norm(x, x.shape[-1:], eps=1e-6) * (1 + scale[:, None]) + shift[:, None]


def _forward64(p, heads):
    t = {n: v.double() for n, v in p.items()}
    b, l, c = t["x"].shape
    s1, t1, g1, s2, t2, g2 = t["mod"].chunk(6, dim=-1)
    d = c // heads
    q, k, v = (_norm64(t["x"], s1, t1) @ t["qkv"].T + t["qkv_b"]).view(b, l, 3, heads, d).unbind(2)
    rope = _rope(l, d).double()

    def turn(u, w):
        u = u / (u.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
        e, o = u[..., 0::2], u[..., 1::2]
        co, si = rope[:, None, :, 0], rope[:, None, :, 1]
        return torch.stack([e * co - o * si, e * si + o * co], dim=-1).flatten(-2)

    q, k = turn(q, t["wq"]), turn(k, t["wk"])
    a = torch.softmax(torch.einsum("blhd,bmhd->bhlm", q, k) * d ** -0.5, dim=-1)
    o = torch.einsum("bhlm,bmhd->blhd", a, v).reshape(b, l, c)
    x = t["x"] + g1[:, None] * (o @ t["proj"].T)
    h = torch.nn.functional.gelu(_norm64(x, s2, t2) @ t["up"].T + t["up_b"], approximate="tanh")
    return x, x + g2[:, None] * (h @ t["down"].T)


@pytest.mark.parametrize("b,l,heads,d", [(1, 1, 2, 128), (2, 77, 4, 64), (2, 300, 6, 128)])
def test_block(b, l, heads, d):
    from dgx_monarch_b200.block_norm import block_norm
    from dgx_monarch_b200.linear import linear
    from dgx_monarch_b200.ops import attention_fwd
    from dgx_monarch_b200.qk_norm import qk_norm_rope

    p = _case(l, b, l, heads, d)
    s1, t1, g1, s2, t2, g2 = p["mod"].chunk(6, dim=-1)
    _, y = block_norm(p["x"], scale=s1, shift=t1)
    qkv = linear(y, p["qkv"], bias=p["qkv_b"])
    q, k, v = qkv.view(b, l, 3, heads, d).unbind(2)
    q, k = qk_norm_rope(q, k, norm_q_w=p["wq"], norm_k_w=p["wk"], rope=_rope(l, d))
    o, _ = attention_fwd(q, k, v)
    branch = linear(o.reshape(b, l, heads * d), p["proj"])
    x, y = block_norm(p["x"], branch, gate=g1, scale=s2, shift=t2)  # the branch joins the stream on the way to the next norm
    fused = linear(o.reshape(b, l, heads * d), p["proj"], gate=g1, residual=p["x"])  # or in the Linear
    h = linear(y, p["up"], bias=p["up_b"], activation="gelu_tanh")
    out = linear(h, p["down"], gate=g2, residual=x)
    want_x, want = _forward64(p, heads)
    assert rel(x, want_x) <= 7 * HALF and rel(fused, want_x) <= 7 * HALF  # y, qkv, q/k, scores, o, branch, x
    assert rel(out, want) <= 10 * HALF  # and y, h, out


@pytest.mark.parametrize("b,l,heads,d", [(1, 1, 2, 128), (2, 77, 4, 64), (2, 300, 6, 128)])
def test_training_step_of_its_second_half(b, l, heads, d):
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward
    from dgx_monarch_b200.linear import linear, linear_backward

    p = _case(l + 1, b, l, heads, d)
    branch = _case(l + 2, b, l, heads, d)["x"]
    _, _, g1, s2, t2, g2 = p["mod"].chunk(6, dim=-1)
    x, y = block_norm(p["x"], branch, gate=g1, scale=s2, shift=t2)
    h, pre_h = linear(y, p["up"], bias=p["up_b"], activation="gelu_tanh", return_pre=True)
    _, pre_o = linear(h, p["down"], gate=g2, residual=x, return_pre=True)
    down = linear_backward(p["dout"], h, p["down"], gate=g2, pre=pre_o)
    up = linear_backward(down.x, y, p["up"], bias=p["up_b"], activation="gelu_tanh", pre=pre_h)
    norm = block_norm_backward(up.x, p["dout"], x, branch, gate=g1, scale=s2, shift=t2)

    leaves = {n: t.double().requires_grad_(True) for n, t in
              (("x", p["x"]), ("branch", branch), ("g1", g1), ("s2", s2), ("t2", t2), ("g2", g2), ("up", p["up"]),
               ("up_b", p["up_b"]), ("down", p["down"]))}
    stream = leaves["x"] + leaves["g1"][:, None] * leaves["branch"]
    hidden = torch.nn.functional.gelu(_norm64(stream, leaves["s2"], leaves["t2"]) @ leaves["up"].T + leaves["up_b"],
                                      approximate="tanh")
    out = stream + leaves["g2"][:, None] * (hidden @ leaves["down"].T)
    out.backward(p["dout"].double())
    # roundings behind each gradient: x, y, pre, h, pre of the forward; dz, dx, dz, dx, and its own
    for name, got in (("down", down.w), ("g2", down.gate), ("up", up.w), ("up_b", up.bias), ("x", norm.x), ("branch", norm.branch),
                      ("g1", norm.gate), ("s2", norm.scale), ("t2", norm.shift)):
        assert rel(got, leaves[name].grad) <= 10 * HALF, (name, rel(got, leaves[name].grad))


def test_block_in_a_graph():
    """Captured together and replayed on new data: the same bits as the calls."""
    from dgx_monarch_b200.block_norm import block_norm
    from dgx_monarch_b200.linear import linear

    p = _case(3, 2, 130, 5, 128)
    _, _, g1, s2, t2, g2 = p["mod"].chunk(6, dim=-1)
    branch = p["dout"].clone()

    def half():
        x, y = block_norm(p["x"], branch, gate=g1, scale=s2, shift=t2)
        return linear(linear(y, p["up"], bias=p["up_b"], activation="gelu"), p["down"], gate=g2, residual=x)

    half()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = half()
    for _ in range(3):
        p["x"].mul_(-0.5)
        branch.add_(0.25)
        graph.replay()
        assert torch.equal(out, half())

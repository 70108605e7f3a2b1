"""The rest of a transformer block around its attention, as cases that can be timed and checked.

Two families, each with its gradient:

* ``norm``: a branch added to the residual stream under a gate (and, with ``post``, an RMSNorm of its own), and the norm of
  the sum with the next branch's scale and shift, in one pass (``block_norm``, ``block_norm_backward``).
* ``linear``: a 16-bit Linear with bias, activation, gate and residual in its epilogue (``linear``, ``linear_backward``).

``run`` computes them in plain torch operations, or through ``dgx_monarch_b200`` where ``own`` is
true.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6
_ACTS = ["none", "silu", "gelu", "gelu_tanh"]


# ------------------------------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # One token before a block of a 5120-wide model: a call whose cost is its latency.
        {"name": "norm_one_token", "op": "norm", "back": False, "batch": 1, "len": 1, "width": 5120, "mode": "layer",
         "affine": False, "branch": False, "gate": False, "post": False, "mod": "sample", "wide_mod": True, "type": "bf16"},
        # One of eight ranks' share of a 75600-token video between two branches of a block.
        {"name": "norm_video_rank", "op": "norm", "back": False, "batch": 1, "len": 9450, "width": 5120, "mode": "layer",
         "affine": False, "branch": True, "gate": True, "post": False, "mod": "sample", "wide_mod": True, "type": "bf16"},
        # Norms before and after a branch, a batch of ragged length, rows that end inside every word.
        {"name": "norm_ragged", "op": "norm", "back": False, "batch": 3, "len": 777, "width": 1365, "mode": "rms",
         "affine": True, "branch": True, "gate": True, "post": True, "mod": "sample", "wide_mod": False, "type": "fp16"},
        # Tokens at different noise levels (image to video): a scale, shift and gate for every token.
        {"name": "norm_token_modulation", "op": "norm", "back": False, "batch": 2, "len": 2640, "width": 2048, "mode": "layer",
         "affine": True, "branch": True, "gate": True, "post": False, "mod": "token", "wide_mod": True, "type": "bf16"},
        # A short text prompt's training step in full precision.
        {"name": "norm_text_gradient", "op": "norm", "back": True, "batch": 2, "len": 77, "width": 1536, "mode": "rms",
         "affine": True, "branch": True, "gate": True, "post": True, "mod": "sample", "wide_mod": False, "type": "fp32"},
        # The training step of the video rank above.
        {"name": "norm_video_gradient", "op": "norm", "back": True, "batch": 1, "len": 9450, "width": 5120, "mode": "layer",
         "affine": False, "branch": True, "gate": True, "post": False, "mod": "sample", "wide_mod": True, "type": "bf16"},
        # Modulation of a block by the conditioning vectors of a batch of two: one pass over the weight.
        {"name": "linear_modulation", "op": "linear", "back": False, "batch": 2, "len": 1, "cols": 5120, "outs": 30720,
         "act": "none", "bias": True, "gate": "none", "residual": False, "type": "bf16"},
        # Sizes that fill no tile and no word, everything in the epilogue.
        {"name": "linear_ragged", "op": "linear", "back": False, "batch": 2, "len": 501, "cols": 1003, "outs": 777,
         "act": "silu", "bias": True, "gate": "sample", "residual": True, "type": "fp16"},
        # The feed-forward expansion of a rank's 9450 tokens.
        {"name": "linear_video_up", "op": "linear", "back": False, "batch": 1, "len": 9450, "cols": 5120, "outs": 13824,
         "act": "gelu_tanh", "bias": True, "gate": "none", "residual": False, "type": "bf16"},
        # And back onto the residual stream, under the block's gate.
        {"name": "linear_video_down", "op": "linear", "back": False, "batch": 1, "len": 9450, "cols": 13824, "outs": 5120,
         "act": "none", "bias": True, "gate": "sample", "residual": True, "type": "bf16"},
        # The text tokens' training step.
        {"name": "linear_text_gradient", "op": "linear", "back": True, "batch": 1, "len": 512, "cols": 4096, "outs": 5120,
         "act": "gelu", "bias": True, "gate": "sample", "residual": False, "type": "fp16"},
        # The training step of the expansion: the largest products of the block.
        {"name": "linear_video_gradient", "op": "linear", "back": True, "batch": 1, "len": 9450, "cols": 5120, "outs": 13824,
         "act": "gelu_tanh", "bias": True, "gate": "none", "residual": False, "type": "bf16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo: int, hi: int) -> int:
    """Whole 64s three times in five, whole 8s or any number else."""
    n, unit = _log(rng, lo, hi), rng.choice([64, 64, 64, 8, 1])
    return min(hi, max(lo, (n + unit - 1) // unit * unit))


def draw(rng) -> dict:
    batch = rng.randint(1, 4)
    if rng.random() < 0.5:
        width, branch = _size(rng, 256, 8192), rng.random() < 0.7
        kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 9450 * 5120 * 2 // (width * batch * _BYTES[kind])
        return {"op": "norm", "back": rng.random() < 0.5, "batch": batch, "len": _log(rng, 1, max(1, min(9450, most))),
                "width": width, "mode": rng.choice(["layer", "rms"]), "affine": rng.random() < 0.5, "branch": branch,
                "gate": branch and rng.random() < 0.8, "post": branch and rng.random() < 0.3,
                "mod": rng.choice(["sample", "sample", "token", "none"]), "wide_mod": rng.random() < 0.5, "type": kind}
    return {"op": "linear", "back": rng.random() < 0.4, "batch": batch, "len": _log(rng, 1, 9450 // batch),
            "cols": _size(rng, 16, 13824), "outs": _size(rng, 8, 5120), "act": rng.choice(_ACTS), "bias": rng.random() < 0.7,
            "gate": rng.choice(["none", "none", "sample", "token"]), "residual": rng.random() < 0.4,
            "type": rng.choice(["bf16", "bf16", "fp16"])}


def work(case: dict) -> dict:
    size, tokens = _BYTES[case["type"]], case["batch"] * case["len"]
    if case["op"] == "norm":
        values = tokens * case["width"]
        both = case["branch"] and (case["gate"] or case["post"])  # otherwise the branch's gradient is the stream's
        if case["back"]:  # the upstream gradients and the stream (and the branch) read, the gradients written
            tensors = 6 if both else 4
        else:
            tensors = 4 if case["branch"] else 2
        held = 4 if case["wide_mod"] else size
        groups = {"none": 0, "sample": case["batch"], "token": tokens}[case["mod"]]
        vectors = groups * (2 + case["gate"]) * (2 if case["back"] else 1)  # scale, shift and gate, and their gradients
        if case["back"]:
            vectors -= groups  # the shift itself is not needed
        if case["gate"] and case["mod"] == "none":
            vectors += (2 if case["back"] else 1) * case["batch"]
        return {"bytes": tensors * values * size + vectors * case["width"] * held, "flops": (30 if case["back"] else 12) * values}
    cols, outs = case["cols"], case["outs"]
    gate = {"none": 0, "sample": case["batch"], "token": tokens}[case["gate"]] * outs
    if case["back"]:  # both operands and the upstream gradient read, both gradients written
        pre = tokens * outs if case["act"] != "none" or case["gate"] != "none" else 0
        return {"bytes": size * (2 * tokens * cols + 2 * outs * cols + tokens * outs + pre + 2 * gate + case["bias"] * outs),
                "flops": 4 * tokens * cols * outs}
    return {"bytes": size * (tokens * cols + outs * cols + tokens * outs * (2 if case["residual"] else 1) + gate + case["bias"] * outs),
            "flops": 2 * tokens * cols * outs}


# ------------------------------------------------------------------------------------- the inputs

def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, batch: int, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """Normal values of differing size by token, with a few channels that stand out."""
    x = _normal(g, batch, rows, cols) * torch.exp(0.5 * _normal(g, batch, rows, 1))
    x = x * (1 + 12 * (torch.rand(cols, device="cuda", generator=g) > 0.995)) + 0.1 * _normal(g, cols)
    return x.to(dtype)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, b, l = _TYPES[case["type"]], case["batch"], case["len"]
    state = {"case": case}
    if case["op"] == "norm":
        c = case["width"]
        held = torch.float32 if case["wide_mod"] else dtype
        state["x"] = _activations(g, b, l, c, dtype)  # the residual stream (gradient: after the branch)
        state["branch"] = _normal(g, b, l, c).mul_(0.7).to(dtype) if case["branch"] else None
        # one projection of the conditioning holds shift, scale and gate side by side
        rows = (b, l) if case["mod"] == "token" else (b,)
        parts = (0.3 * _normal(g, *rows, 3 * c)).to(held).chunk(3, dim=-1)
        state["shift"], state["scale"] = parts[:2] if case["mod"] != "none" else (None, None)
        state["gate"] = parts[2] if case["gate"] else None
        state["norm_w"] = (1 + 0.2 * _normal(g, c)).to(dtype) if case["affine"] else None
        state["norm_b"] = (0.2 * _normal(g, c)).to(dtype) if case["affine"] and case["mode"] == "layer" else None
        state["branch_w"] = (1 + 0.2 * _normal(g, c)).to(dtype) if case["post"] else None
        if case["back"]:
            state["dy"], state["dr"] = _normal(g, b, l, c).to(dtype), _normal(g, b, l, c).to(dtype)
        return state
    k, n = case["cols"], case["outs"]
    state["x"] = _activations(g, b, l, k, dtype)
    state["w"] = (_normal(g, n, k) * k ** -0.5).to(dtype)
    state["bias"] = (0.2 * _normal(g, n)).to(dtype) if case["bias"] else None
    state["gate"] = None
    if case["gate"] != "none":
        state["gate"] = (0.5 * _normal(g, *((b, l, n) if case["gate"] == "token" else (b, n)))).to(dtype)
    if case["back"]:
        needs = case["act"] != "none" or case["gate"] != "none"
        pre = state["x"] @ state["w"].T if needs else None  # what the forward pass kept
        state["pre"] = pre if pre is None or state["bias"] is None else pre + state["bias"]
        state["dout"] = _normal(g, b, l, n).to(dtype)
    else:
        state["residual"] = _activations(g, b, l, n, dtype) if case["residual"] else None
    return state


# ------------------------------------------------------------------------------------- plain forms

def _rows(t: torch.Tensor | None, back: bool = False):
    """A modulation in 32 bits against (batch, rows, values): one for each token, or one for each sample."""
    if t is None:
        return None
    return t.float() if t.ndim == 3 else t.float()[:, None]


def _plain_norm(s: dict, case: dict) -> list:
    r, w2 = s["x"].float(), s["branch_w"]
    if case["branch"]:
        m = s["branch"].float()
        if case["post"]:
            m = m * torch.rsqrt((m * m).mean(-1, keepdim=True) + _EPS) * w2.float()
        r = r + (m if s["gate"] is None else _rows(s["gate"]) * m)
    n = r - r.mean(-1, keepdim=True) if case["mode"] == "layer" else r
    y = n * torch.rsqrt((n * n).mean(-1, keepdim=True) + _EPS)
    if s["norm_w"] is not None:
        y = y * s["norm_w"].float()
    if s["norm_b"] is not None:
        y = y + s["norm_b"].float()
    if s["scale"] is not None:
        y = y * (1 + _rows(s["scale"])) + _rows(s["shift"])
    dtype = s["x"].dtype
    return [r.to(dtype), y.to(dtype)] if case["branch"] else [y.to(dtype)]


def _summed(values: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """The gradient of a modulation: over its sample's rows, or the token's own."""
    return (values if like.ndim == 3 else values.sum(1)).to(like.dtype)


def _plain_norm_backward(s: dict, case: dict) -> list:
    dtype, dy = s["x"].dtype, s["dy"].float()
    n = s["x"].float()
    if case["mode"] == "layer":
        n = n - n.mean(-1, keepdim=True)
    rstd = torch.rsqrt((n * n).mean(-1, keepdim=True) + _EPS)
    n = n * rstd
    h = n if s["norm_w"] is None else n * s["norm_w"].float()
    if s["norm_b"] is not None:
        h = h + s["norm_b"].float()
    dscale = dshift = dgate = dw = db = dw2 = None
    dh = dy
    if s["scale"] is not None:
        dshift, dscale = _summed(dy, s["shift"]), _summed(dy * h, s["scale"])
        dh = dy * (1 + _rows(s["scale"]))
    dn = dh
    if s["norm_w"] is not None:
        dw = (dh * n).sum((0, 1)).to(dtype)
        dn = dh * s["norm_w"].float()
    if s["norm_b"] is not None:
        db = dh.sum((0, 1)).to(dtype)
    inner = dn - n * (dn * n).mean(-1, keepdim=True)
    if case["mode"] == "layer":
        inner = inner - dn.mean(-1, keepdim=True)
    dr = s["dr"].float() + rstd * inner
    dx, dbranch = dr.to(dtype), None
    if case["branch"]:
        m, dm = s["branch"].float(), dr
        if case["post"]:
            w2 = s["branch_w"].float()
            rstd2 = torch.rsqrt((m * m).mean(-1, keepdim=True) + _EPS)
            n2 = m * rstd2
            m = n2 * w2
        if s["gate"] is not None:
            dgate = _summed(dr * m, s["gate"])
            dm = dr * _rows(s["gate"])
        if case["post"]:
            dw2 = (dm * n2).sum((0, 1)).to(dtype)
            dn2 = dm * w2
            dm = rstd2 * (dn2 - n2 * (dn2 * n2).mean(-1, keepdim=True))
        dbranch = dm.to(dtype)
    return [t for t in (dx, dbranch, dgate, dw2, dw, db, dscale, dshift) if t is not None]


def _act(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 2 ** -0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 2 ** -0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    u = (2 / math.pi) ** 0.5
    t = torch.tanh(u * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * u * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s: dict, case: dict) -> list:
    z = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["act"])
    if s["gate"] is not None:
        y = y * _rows(s["gate"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return [y.to(s["x"].dtype)]


def _plain_linear_backward(s: dict, case: dict) -> list:
    dtype, dout = s["x"].dtype, s["dout"].float()
    dz, dgate = dout, None
    if s["gate"] is not None:
        dgate = _summed(dout * _act(s["pre"].float(), case["act"]), s["gate"])
        dz = dout * _rows(s["gate"])
    if case["act"] != "none":
        dz = dz * _act_slope(s["pre"].float(), case["act"])
    flat = dz.flatten(0, 1)
    dx, dw = dz @ s["w"].float(), flat.T @ s["x"].float().flatten(0, 1)
    got = [dx.to(dtype), dw.to(dtype)]
    if s["bias"] is not None:
        got.append(flat.sum(0).to(dtype))
    return got if dgate is None else got + [dgate]


# ------------------------------------------------------------------------------------- one pass

def run(state: dict):
    case = state["case"]
    if not own:
        if case["op"] == "norm":
            return _plain_norm_backward(state, case) if case["back"] else _plain_norm(state, case)
        return _plain_linear_backward(state, case) if case["back"] else _plain_linear(state, case)
    s = state
    if case["op"] == "norm":
        from dgx_monarch_b200.block_norm import NORM_LAYER, NORM_RMS, block_norm, block_norm_backward

        keep = {"gate": s["gate"], "branch_norm": case["post"], "branch_w": s["branch_w"],
                "norm_mode": NORM_LAYER if case["mode"] == "layer" else NORM_RMS, "norm_w": s["norm_w"], "norm_b": s["norm_b"],
                "scale": s["scale"], "shift": s["shift"], "eps": _EPS}
        if case["back"]:
            grads = block_norm_backward(s["dy"], s["dr"], s["x"], s["branch"], **keep)
            return [t for t in (grads.x, grads.branch, grads.gate, grads.branch_w, grads.norm_w, grads.norm_b, grads.scale,
                                grads.shift) if t is not None]
        r, y = block_norm(s["x"], s["branch"], **keep)
        return [r, y] if case["branch"] else [y]
    from dgx_monarch_b200.linear import linear, linear_backward

    if case["back"]:
        grads = linear_backward(s["dout"], s["x"], s["w"], bias=s["bias"], activation=case["act"], gate=s["gate"], pre=s["pre"])
        return [t for t in (grads.x, grads.w, grads.bias, grads.gate) if t is not None]
    return [linear(s["x"], s["w"], bias=s["bias"], activation=case["act"], gate=s["gate"], residual=s["residual"])]


# ------------------------------------------------------------------------------------- in 64 bits

def _double(t: torch.Tensor | None, grad: bool = False):
    return None if t is None else t.detach().double().requires_grad_(grad)


def _exact_act(z: torch.Tensor, name: str) -> torch.Tensor:
    f = torch.nn.functional
    return {"none": lambda v: v, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[name](z)


def _exact_branch(branch, gate, w2, post: bool):
    """What the branch adds to the stream."""
    m = torch.nn.functional.rms_norm(branch, branch.shape[-1:], w2, _EPS) if post else branch
    return m if gate is None else m * (gate if gate.ndim == 3 else gate.unsqueeze(1))


def _exact_normed(r, w, b, scale, shift, mode: str):
    f, c = torch.nn.functional, r.shape[-1:]
    h = f.layer_norm(r, c, w, b, _EPS) if mode == "layer" else f.rms_norm(r, c, w, _EPS)
    if scale is None:
        return h
    lift = (lambda t: t) if scale.ndim == 3 else (lambda t: t.unsqueeze(1))
    return torch.addcmul(h + lift(shift), h, lift(scale))


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    back = case["back"]
    if case["op"] == "norm":
        names = ("x", "branch", "gate", "branch_w", "norm_w", "norm_b", "scale", "shift")
        v = {n: _double(s[n], back) for n in names}
        r = v["x"]
        if case["branch"]:
            added = _exact_branch(v["branch"], v["gate"], v["branch_w"], case["post"])
            # the gradient's stream already holds the branch
            r = r + (added - added.detach() if back else added)
        y = _exact_normed(r, v["norm_w"], v["norm_b"], v["scale"], v["shift"], case["mode"])
        if not back:
            return [r, y] if case["branch"] else [y]
        leaves = [v[n] for n in names if v[n] is not None]
        return list(torch.autograd.grad([y, r], leaves, [s["dy"].double(), s["dr"].double()]))
    x, w, bias, gate = (s[n].double() if s[n] is not None else None for n in ("x", "w", "bias", "gate"))
    if gate is not None and gate.ndim == 2:
        gate = gate.unsqueeze(1)
    if not back:
        y = _exact_act(torch.nn.functional.linear(x, w, bias), case["act"])
        y = y if gate is None else y * gate
        return [y if s["residual"] is None else y + s["residual"].double()]
    dz, dgate = s["dout"].double(), None
    if s["pre"] is not None:
        pre = _double(s["pre"], True)
        held = None if gate is None else gate.requires_grad_(True)
        y = _exact_act(pre, case["act"])
        y = y if held is None else y * held
        got = torch.autograd.grad(y, [pre] if held is None else [pre, held], dz)
        dz = got[0]
        if held is not None:
            dgate = got[1] if s["gate"].ndim == 3 else got[1].squeeze(1)
        del y, pre
    out = [torch.einsum("bln,nk->blk", dz, w), torch.einsum("bln,blk->nk", dz, x)]
    if bias is not None:
        out.append(torch.einsum("bln->n", dz))
    return out if dgate is None else out + [dgate]

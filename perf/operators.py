"""Operators around the attention of a transformer block, as cases that can be timed and checked.

Two families:

* ``qk``: RMSNorm of every query and key head with the rotary position embedding in the same
  pass (``qk_norm_rope``), and its gradient (``qk_norm_rope_backward``).
* ``quant`` and ``linear``: microscaled 4-bit floating point (e2m1 values; nvfp4: one e4m3 scale
  for 16 values and one fp32 scale for the tensor; mxfp4: one power of two for 32 values), written
  and read back, and the product of two such tensors (``quantize_fp4``, ``dequantize_fp4``,
  ``fp4_matmul``).

``run`` computes them in plain torch operations, or through ``dgx_monarch_b200`` where ``own`` is
true.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BLOCK = {"nvfp4": 16, "mxfp4": 32}
_EPS = 1e-6


# ------------------------------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # One token of a 40-head model: a call whose cost is its latency.
        {"name": "qk_one_token", "op": "qk", "back": False, "batch": 1, "len": 1, "q_heads": 40, "k_heads": 40,
         "dim": 128, "rot": 128, "halves": False, "norm": True, "type": "bf16"},
        # One of eight ranks' share of a 75600-token video, 40 heads: the ordinary call of a sequence-parallel step.
        {"name": "qk_video_rank", "op": "qk", "back": False, "batch": 1, "len": 9450, "q_heads": 40, "k_heads": 40,
         "dim": 128, "rot": 128, "halves": False, "norm": True, "type": "bf16"},
        # Shared key heads, a ragged length, an odd head size of which only a part is rotated, halves rotated against each other.
        {"name": "qk_grouped_ragged", "op": "qk", "back": False, "batch": 3, "len": 777, "q_heads": 20, "k_heads": 4,
         "dim": 96, "rot": 64, "halves": True, "norm": True, "type": "fp16"},
        # A short text prompt's training step in full precision.
        {"name": "qk_text_gradient", "op": "qk", "back": True, "batch": 2, "len": 77, "q_heads": 8, "k_heads": 8,
         "dim": 64, "rot": 64, "halves": False, "norm": True, "type": "fp32"},
        # The training step of the video rank above.
        {"name": "qk_video_gradient", "op": "qk", "back": True, "batch": 1, "len": 9450, "q_heads": 40, "k_heads": 40,
         "dim": 128, "rot": 128, "halves": False, "norm": True, "type": "bf16"},
        # The conditioning vector of one sample, with the scale that the ranks share.
        {"name": "quant_one_row", "op": "quant", "rows": 1, "cols": 5120, "format": "nvfp4", "given": True, "type": "bf16"},
        # The activations of a rank's 9450 tokens, the tensor's scale found on the way.
        {"name": "quant_video_rank", "op": "quant", "rows": 9450, "cols": 5120, "format": "nvfp4", "given": False, "type": "bf16"},
        # Odd rows and columns, blocks of 32 that the last columns do not fill.
        {"name": "quant_ragged_mx", "op": "quant", "rows": 1003, "cols": 2731, "format": "mxfp4", "given": False, "type": "fp16"},
        # Modulation of a block by the conditioning vectors of a batch of two: one pass over the weight.
        {"name": "linear_modulation", "op": "linear", "rows": 2, "cols": 5120, "outs": 30720, "format": "nvfp4", "packed": False,
         "bias": True, "given": True, "type": "bf16"},
        # The text tokens' projection.
        {"name": "linear_text", "op": "linear", "rows": 512, "cols": 5120, "outs": 5120, "format": "mxfp4", "packed": False,
         "bias": True, "given": False, "type": "fp16"},
        # Both operands at hand in 4 bits, sizes that fill no tile.
        {"name": "linear_ragged_packed", "op": "linear", "rows": 1003, "cols": 1000, "outs": 777, "format": "nvfp4", "packed": True,
         "bias": False, "given": True, "type": "bf16"},
        # The feed-forward expansion of a rank's 9450 tokens: the largest product of the block.
        {"name": "linear_video_rank", "op": "linear", "rows": 9450, "cols": 5120, "outs": 13824, "format": "nvfp4", "packed": False,
         "bias": True, "given": True, "type": "bf16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["qk", "qk", "quant", "linear", "linear"])
    if op == "qk":
        batch, k_heads = rng.randint(1, 4), rng.choice([1, 2, 4, 5, 8, 10])
        dim = rng.choice([40, 64, 72, 96, 128, 128, 256])
        q_heads = k_heads * rng.choice([1, 1, 2, 4])
        most = max(1, 9450 * 40 * 128 * 2 // (batch * (q_heads + k_heads) * dim * 2))
        return {"op": "qk", "back": rng.random() < 0.5, "batch": batch, "len": _log(rng, 1, min(9450, most)), "q_heads": q_heads,
                "k_heads": k_heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "halves": rng.random() < 0.5,
                "norm": rng.random() < 0.85, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    form = rng.choice(["nvfp4", "mxfp4"])
    given = form == "nvfp4" and rng.random() < 0.5
    if op == "quant":
        cols = _log(rng, 16, 13824)
        return {"op": "quant", "rows": _log(rng, 1, 9450 * 5120 // max(cols, 5120)), "cols": cols, "format": form, "given": given,
                "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    return {"op": "linear", "rows": _log(rng, 1, 9450), "cols": _log(rng, 16, 5120), "outs": _log(rng, 8, 13824), "format": form,
            "packed": rng.random() < 0.3, "bias": rng.random() < 0.5, "given": given, "type": rng.choice(["bf16", "bf16", "fp16"])}


def work(case: dict) -> dict:
    if case["op"] == "qk":
        size = _BYTES[case["type"]]
        tokens = case["batch"] * case["len"]
        values = tokens * (case["q_heads"] + case["k_heads"]) * case["dim"]
        table = case["len"] * case["rot"] // 2 * 8
        if case["back"]:  # the upstream gradient and the inputs read, the inputs' gradient written
            return {"bytes": 3 * values * size + table + 4 * case["dim"] * size, "flops": 14 * values}
        return {"bytes": 2 * values * size + table + 2 * case["dim"] * size, "flops": 8 * values}
    block = _BLOCK[case["format"]]
    held = 0.5 + 1.0 / block  # bytes of one value in 4 bits with its share of the scale
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "quant":  # the values read, written in 4 bits, read, and written back
        return {"bytes": rows * cols * (2 * _BYTES[case["type"]] + 2 * held), "flops": 4 * rows * cols}
    outs = case["outs"]
    x = rows * cols * (held if case["packed"] else 2)
    return {"bytes": x + outs * cols * held + rows * outs * 2 + (2 * outs if case["bias"] else 0), "flops": 2 * rows * cols * outs}


# ------------------------------------------------------------------------------------- the inputs

def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _angles(case: dict) -> torch.Tensor:
    """(len, rot / 2) angles in 64 bits of a video's (t, h, w) positions: the pairs split over the three axes."""
    pairs = case["rot"] // 2
    at = torch.arange(case["len"], device="cuda", dtype=torch.float64)
    axis = torch.arange(pairs, device="cuda") * 3 // max(1, pairs)
    omega = 10000.0 ** -((torch.arange(pairs, device="cuda", dtype=torch.float64) * 3 % max(1, pairs)) / max(1, pairs))
    place = torch.stack([torch.floor(at / 1560), torch.floor(at / 52) % 30, at % 52], dim=1)
    return place[:, axis] * omega


def _activations(g, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """Normal values of differing size by token, with a few channels that stand out."""
    x = _normal(g, rows, cols) * torch.exp(0.5 * _normal(g, rows, 1))
    x = x * (1 + 12 * (torch.rand(cols, device="cuda", generator=g) > 0.995))
    return x.to(dtype)


def _stored(x: torch.Tensor, form: str) -> dict:
    """A weight in 4 bits as the framework's files and users hold it: two values a byte, the first in the low bits, rows of whole
    16 bytes; scale bytes by tiles of 128 rows x 4 blocks as (row tile, block group, row % 32, row % 128 // 32, block % 4)."""
    block, (rows, cols) = _BLOCK[form], x.shape
    values, scale_bytes, scale = _to_4_bits(x, form, None)
    pitch = (cols + 31) // 32 * 16
    code = torch.zeros(rows, 2 * pitch, device="cuda", dtype=torch.uint8)
    code[:, :cols] = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device="cuda", dtype=torch.uint8)[(values.abs() * 2).long()]
    code[:, :cols] |= torch.signbit(values).to(torch.uint8) << 3
    tiles, groups = (rows + 127) // 128, ((cols + block - 1) // block + 3) // 4
    at = torch.zeros(tiles * 128, groups * 4, device="cuda", dtype=torch.uint8)
    at[:rows, :scale_bytes.shape[1]] = scale_bytes
    at = at.view(tiles, 4, 32, groups, 4).permute(0, 3, 2, 1, 4).contiguous()
    return {"values": code[:, 0::2] | code[:, 1::2] << 4, "scales": at, "scale": scale, "shape": (rows, cols), "format": form}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["type"]]
    if case["op"] == "qk":
        b, l, hq, hk, d = case["batch"], case["len"], case["q_heads"], case["k_heads"], case["dim"]
        # q and k are views of one projection's output, next to v
        qkv = (_normal(g, b, l, hq + 2 * hk, d) * torch.exp(0.5 * _normal(g, b, l, 1, 1))).to(dtype)
        angle = _angles(case)
        state = {"case": case, "q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk],
                 "wq": (1 + 0.2 * _normal(g, d)).to(dtype) if case["norm"] else None,
                 "wk": (1 + 0.2 * _normal(g, d)).to(dtype) if case["norm"] else None,
                 "rope": torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1).float()}
        if case["back"]:
            state["dq"], state["dk"] = _normal(g, b, l, hq, d).to(dtype), _normal(g, b, l, hk, d).to(dtype)
        return state
    state = {"case": case}
    x = _activations(g, case["rows"], case["cols"], dtype)
    given = None
    if case["given"]:  # the scale that the ranks have agreed on, in the activations' type
        given = (x.abs().amax().float() / 2688).to(dtype)
    if case["op"] == "linear":
        w = _normal(g, case["outs"], case["cols"]) * case["cols"] ** -0.5
        state["w"] = _stored(w, case["format"])
        state["bias"] = _normal(g, case["outs"]).to(dtype) if case["bias"] else None
        if case["packed"]:
            state["a"] = _stored(x, case["format"])
            return state
    state["x"], state["given"] = x, given
    return state


# ------------------------------------------------------------------------------------- plain forms

def _rotate(y: torch.Tensor, rope: torch.Tensor, rot: int, halves: bool, back: bool) -> torch.Tensor:
    c, s = rope[..., 0][:, None], rope[..., 1][:, None]
    if back:
        s = -s
    z, r = y[..., :rot], rot // 2
    a, b = (z[..., :r], z[..., r:]) if halves else (z[..., 0::2], z[..., 1::2])
    u, v = a * c - b * s, a * s + b * c
    turned = torch.cat([u, v], dim=-1) if halves else torch.stack([u, v], dim=-1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], dim=-1)


def _norm_rotate(x, w, rope, case):
    y = x.float()
    if case["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * w.float()
    return _rotate(y, rope, case["rot"], case["halves"], False).to(x.dtype)


def _norm_rotate_back(dy, x, w, rope, case):
    g = _rotate(dy.float(), rope, case["rot"], case["halves"], True)
    if not case["norm"]:
        return g.to(x.dtype), None
    y = x.float()
    r = torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS)
    n = y * r
    dw = (g * n).sum((0, 1, 2))
    g = g * w.float()
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype), dw.to(w.dtype)


def _step(x: torch.Tensor, least: int, bits: int) -> torch.Tensor:
    """The distance of neighbouring values of a float format around |x|, in 64 bits."""
    e = torch.frexp(x.abs())[1] - 1
    return torch.ldexp(torch.ones_like(x), e.clamp(min=least) - bits)


def _blocks(x: torch.Tensor, block: int) -> torch.Tensor:
    pad = -x.shape[1] % block
    return torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], -1, block)


def _to_4_bits(x, form: str, given):
    """(e2m1 values, scale bytes, tensor scale) of a matrix, the borders decided in 64 bits."""
    rows, cols = x.shape
    v = _blocks(x, _BLOCK[form]).double()
    most = v.abs().amax(-1)
    if form == "nvfp4":
        scale = given.float() if given is not None else (x.abs().amax().double() / 2688).float()
        t = most / (6 * scale.double())
        t = t.clamp(max=448.0)
        step = _step(t, -6, 3)
        s = (torch.round(t / step) * step).clamp(max=448.0)
        scale_bytes = s.float().to(torch.float8_e4m3fn).view(torch.uint8)
        unit = s * scale.double()
    else:
        scale = None
        e = torch.where(most > 0, torch.frexp(most)[1] - 3, -127).clamp(-127, 127)
        scale_bytes = (e + 127).to(torch.uint8)
        unit = torch.ldexp(torch.ones_like(most), e)
    t = torch.where(unit[..., None] > 0, v / unit[..., None], 0.0).clamp(-6.0, 6.0)
    step = _step(t, 0, 1)
    return (torch.round(t / step) * step).reshape(rows, -1)[:, :cols].float(), scale_bytes, scale


def _scaled(values, scale_bytes, scale, form: str) -> torch.Tensor:
    """The values in 32 bits that 4-bit ones with their scales stand for."""
    block = _BLOCK[form]
    if form == "nvfp4":
        s = scale_bytes.view(torch.float8_e4m3fn).float()
    else:
        s = torch.ldexp(torch.ones_like(scale_bytes, dtype=torch.float32), scale_bytes.int() - 127)
    out = values * s.repeat_interleave(block, dim=1)[:, :values.shape[1]]
    return out if scale is None else out * scale


def _loaded(t: dict) -> torch.Tensor:
    rows, cols = t["shape"]
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    code = torch.stack([t["values"] & 15, t["values"] >> 4], dim=-1).view(rows, -1)[:, :cols]
    tiles, groups = t["scales"].shape[:2]
    at = t["scales"].permute(0, 3, 2, 1, 4).reshape(tiles * 128, groups * 4)[:rows, :-(-cols // _BLOCK[t["format"]])]
    return _scaled(table[code.int()], at.contiguous(), t["scale"], t["format"])


def _run_plain(state):
    case = state["case"]
    if case["op"] == "qk":
        if not case["back"]:
            return [_norm_rotate(state["q"], state["wq"], state["rope"], case), _norm_rotate(state["k"], state["wk"], state["rope"], case)]
        gq, gwq = _norm_rotate_back(state["dq"], state["q"], state["wq"], state["rope"], case)
        gk, gwk = _norm_rotate_back(state["dk"], state["k"], state["wk"], state["rope"], case)
        return [gq, gk] + ([gwq, gwk] if case["norm"] else [])
    form = case["format"]
    if case["op"] == "quant":
        return _scaled(*_to_4_bits(state["x"], form, state["given"]), form).to(state["x"].dtype)
    a = _loaded(state["a"]) if case["packed"] else _scaled(*_to_4_bits(state["x"], form, state["given"]), form)
    y = a @ _loaded(state["w"]).T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(_TYPES[case["type"]])


def _run_own(state):
    from dgx_monarch_b200 import _lib
    from dgx_monarch_b200.fp4 import Fp4Tensor, dequantize_fp4, fp4_matmul, quantize_fp4
    from dgx_monarch_b200.qk_norm import qk_norm_rope, qk_norm_rope_backward

    case = state["case"]
    if case["op"] == "qk":
        how = {"norm_mode": _lib.NORM_HEAD if case["norm"] else _lib.NORM_NONE, "norm_q_w": state["wq"], "norm_k_w": state["wk"],
               "eps": _EPS, "rope": state["rope"], "rope_halves": case["halves"]}
        if not case["back"]:
            return list(qk_norm_rope(state["q"], state["k"], **how))
        got = qk_norm_rope_backward(state["dq"], state["dk"], state["q"], state["k"], **how)
        return list(got) if case["norm"] else list(got[:2])
    dtype = _TYPES[case["type"]]
    if case["op"] == "quant":
        return dequantize_fp4(quantize_fp4(state["x"], format=case["format"], scale=state["given"]), dtype)
    a = Fp4Tensor(**state["a"]) if case["packed"] else quantize_fp4(state["x"], format=case["format"], scale=state["given"])
    return fp4_matmul(a, Fp4Tensor(**state["w"]), bias=state["bias"], out_dtype=dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------- in 64 bits

def _exact_turn(y, rope, case):
    """Rotation as a product of complex numbers."""
    rot, r = case["rot"], case["rot"] // 2
    turn = torch.view_as_complex(rope.double().contiguous())[:, None]
    z = y[..., :rot].unflatten(-1, (2, r)).transpose(-1, -2) if case["halves"] else y[..., :rot].unflatten(-1, (r, 2))
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z.transpose(-1, -2).flatten(-2) if case["halves"] else z.flatten(-2)
    return torch.cat([z, y[..., rot:]], dim=-1)


def _exact_qk(x, w, rope, case):
    if case["norm"]:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w
    return _exact_turn(x, rope, case)


def _exact_codes(x, form, given):
    """The 64-bit values that the 4-bit form stands for: each value goes to the nearest of the format, ties to the even code."""
    block, (rows, cols) = _BLOCK[form], x.shape
    v = _blocks(x.double(), block)
    most = v.abs().max(dim=-1).values
    if form == "nvfp4":
        scale = given.float().double() if given is not None else (x.double().abs().max() / 2688).float().double()
        small = torch.arange(8, device=x.device, dtype=torch.float64) / 8 / 64
        normal = torch.arange(8, 16, device=x.device, dtype=torch.float64) / 8
        grid = torch.cat([small] + [normal * 2.0 ** e for e in range(-6, 9)])[:127]
        unit = _nearest(most / (6 * scale), grid) * scale
    else:
        unit = torch.exp2(torch.clamp(torch.floor(torch.log2(most)) - 2, -127, 127))  # 2^e is exact in 64 bits
        unit = torch.where(unit * 8 <= most, unit * 2, unit)                            # log2 may miss by a step at a power of two
        unit = torch.where(unit * 4 > most, unit / 2, unit).clamp(2.0 ** -127, 2.0 ** 127)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=x.device, dtype=torch.float64)
    unit = unit[..., None]
    t = torch.where(unit > 0, v.abs() / unit.clamp(min=1e-300), 0.0)
    return (torch.copysign(_nearest(t, grid), v) * unit).reshape(rows, -1)[:, :cols]


def _nearest(t, grid):
    at = torch.bucketize(t, grid).clamp(max=len(grid) - 1)  # grid[at - 1] < t <= grid[at], the last one beyond the end
    low = (at - 1).clamp(min=0)
    below, above = t - grid[low], grid[at] - t
    up = (above < below) | ((above == below) & (at % 2 == 0))
    return torch.where(up, grid[at], grid[low])


def _exact_loaded(t):
    rows, cols = t["shape"]
    code = torch.stack([t["values"] % 16, t["values"] // 16], dim=-1).reshape(rows, -1)[:, :cols].long()
    e, m = code % 8 // 2, code % 2
    v = torch.where(e > 0, (1 + m / 2.0) * 2.0 ** (e - 1).double(), m / 2.0) * (1 - 2 * (code // 8))
    block = _BLOCK[t["format"]]
    r = torch.arange(rows, device="cuda")[:, None]
    b = (torch.arange(cols, device="cuda") // block)[None]
    s = t["scales"][r // 128, b // 4, r % 32, r % 128 // 32, b % 4].long()
    if t["format"] == "mxfp4":
        return v * 2.0 ** (s - 127).double()
    e, m = s // 8, (s % 8).double()
    s = torch.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7).double(), m / 8 * 2.0 ** -6)
    return v * s * t["scale"].double()


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "qk":
        got, weights = [], []
        for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
            v = state[x].double().requires_grad_(case["back"])
            u = state[w].double().requires_grad_(case["back"]) if case["norm"] else None
            y = _exact_qk(v, u, state["rope"], case)
            if not case["back"]:
                got.append(y)
                continue
            grads = torch.autograd.grad(y, [v] if u is None else [v, u], state[dy].double())
            got.append(grads[0])
            weights += grads[1:]
        return got + weights
    if case["op"] == "quant":
        return _exact_codes(state["x"], case["format"], state["given"])
    a = _exact_loaded(state["a"]) if case["packed"] else _exact_codes(state["x"], case["format"], state["given"])
    y = a @ _exact_loaded(state["w"]).T
    return y if state["bias"] is None else y + state["bias"].double()

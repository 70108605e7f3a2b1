"""Microscaled 4-bit quantisation and its reading back, bit for bit against
the definitions in 64 bits.

The quotients that decide a rounding are compared in float64 without error:
a border times a block scale times g has at most 3 + 4 + 24 significant bits,
so a float64 quotient equals a border exactly where the real one does, and
lies on the same side of it everywhere else (31 bits apart at the least,
against 53)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from dgx_monarch_b200.fp4 import BLOCK, Fp4Tensor, dequantize_fp4, quantize_fp4

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def _nearest(t, grid):
    """Index of the nearest grid value, ties to the even index, saturating."""
    mid = (grid[1:] + grid[:-1]) / 2
    lo = np.searchsorted(mid, t, side="left")   # a tie stays below
    hi = np.searchsorted(mid, t, side="right")  # a tie goes above
    return np.where(lo % 2 == 0, lo, hi)


def _reference(x, fmt, g):
    """(codes (rows, cols), scale bytes (rows, blocks), values) of a float64 matrix."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    nb = -(-cols // block)
    v = np.zeros((rows, nb * block))
    v[:, :cols] = x
    v = v.reshape(rows, nb, block)
    most = np.abs(v).max(-1)
    broken = ~np.isfinite(most)
    v, most = np.where(broken[..., None], 0, v), np.where(broken, 0, most)
    if fmt == "nvfp4":
        if not (np.isfinite(g) and g >= 0):
            broken, g = np.ones_like(broken), 1.0
        byte = _nearest(most / (6 * g), E4M3) if g > 0 else np.zeros(most.shape, int)
        unit = E4M3[byte] * g
        nan = 0x7F
    else:
        e = np.clip(np.frexp(most)[1] - 3, -127, 127)
        byte = np.where(most > 0, e + 127, 0)
        unit = 2.0 ** (byte.astype(float) - 127)
        nan = 0xFF
    on = (unit > 0) & ~broken
    t = np.where(on[..., None], np.abs(v) / np.where(on, unit, 1)[..., None], 0)
    code = _nearest(t, E2M1)
    val = np.where(broken[..., None], np.nan, np.where(np.signbit(v), -1, 1) * E2M1[code] * unit[..., None])
    code = np.where(on[..., None], code | (np.signbit(v) << 3), 0)
    byte = np.where(broken, nan, byte)
    return code.reshape(rows, -1)[:, :cols], byte, val.reshape(rows, -1)[:, :cols]


def _unpack(t: Fp4Tensor):
    v = t.values.cpu().numpy()
    code = np.stack([v & 15, v >> 4], -1).reshape(t.rows, -1)
    s = t.scales.cpu().numpy().transpose(0, 3, 2, 1, 4).reshape(t.scales.shape[0] * 128, -1)[:t.rows]
    return code, s


def _check(x, fmt, given=None, dtypes=(F32,)):
    t = quantize_fp4(x, format=fmt, scale=given)
    x64 = x.detach().reshape(-1, x.shape[-1]).double().cpu().numpy()
    g = 1.0
    if fmt == "nvfp4":
        if given is None:
            want = (torch.as_tensor(np.abs(x64).max() if x64.size else 0.0) / 2688).float()
        else:
            want = given.float().cpu() if isinstance(given, torch.Tensor) else torch.tensor(given, dtype=F32)
        assert torch.equal(t.scale.cpu().reshape(()), want.reshape(())) or (t.scale.isnan() and want.isnan())
        g = float(want)
    code, byte, val = _reference(x64, fmt, g)
    got_code, got_byte = _unpack(t)
    nb = byte.shape[1]
    assert (got_byte[:, :nb] == byte).all(), np.argwhere(got_byte[:, :nb] != byte)[:5]
    assert (got_byte[:, nb:] == 0).all()
    assert (got_code[:, :t.cols] == code).all(), np.argwhere(got_code[:, :t.cols] != code)[:5]
    assert (got_code[:, t.cols:] == 0).all()
    for dtype in dtypes:
        back = dequantize_fp4(t, dtype)
        assert back.shape == x.shape and back.dtype == dtype
        # code * s is exact; one rounding for g, one to a 16-bit type (in fp32's range here)
        want = torch.from_numpy(val).float().to(dtype).reshape(x.shape)
        assert torch.equal(torch.nan_to_num(back.cpu(), 12345.0), torch.nan_to_num(want, 12345.0))
        assert torch.equal(back.cpu().isnan(), want.isnan())
    return t


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 17), (127, 31), (128, 33), (129, 64), (5, 65), (300, 100),
                                       (2, 5120), (33, 1023), (260, 128), (1, 13824), (300, 1000), (257, 2050)])
def test_sizes(fmt, dtype, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=g))
    _check(x.to(dtype), fmt, dtypes=(F32, dtype))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("amax", [2.0, 3.0, 5.25, 7.0, 2.625, 1.3125])
def test_own_scale_with_borders_beside_values(dtype, amax):
    """g = amax / 2688: where amax s b has the factor 21, a border misses a
    value by the rounding of g alone.  Values around every border of every
    block scale, and the values next to them in their type."""
    gen = torch.Generator(device="cuda").manual_seed(21)
    x = torch.randn(64, 1024, device="cuda", generator=gen) * amax / 4
    lead = amax * torch.arange(1, 65, device="cuda") / 64           # each block's largest, hence its scale
    x = x.clamp(-amax, amax).view(64, 64, 16)
    x = torch.minimum(torch.maximum(x, -lead[:, None]), lead[:, None])
    x[..., 0] = lead
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda") / 6
    x[..., 1:8] = (lead[:, None] * border).to(dtype).float()
    x[..., 8:15] = -x[..., 1:8] * (1 + torch.randint(-2, 3, (64, 64, 7), device="cuda", generator=gen)
                                  * float(torch.finfo(dtype).eps))
    x = x.reshape(64, 1024).to(dtype)
    x[0, 0] = amax
    _check(x, "nvfp4")
    _check(x, "nvfp4", float(x.abs().max()) / 2688)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("g", [1.0, 0.25, 0.3, 0.0078125, 1 / 2688])
def test_given_scale_and_ties(dtype, g):
    """Values on a coarse grid: many quotients lie exactly on a border, and with g not a power of two next to one."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randint(-96, 97, (64, 512), device="cuda", generator=gen).float() / 16
    x *= torch.randint(1, 8, (64, 32, 1), device="cuda", generator=gen).float().expand(64, 32, 16).reshape(64, 512)
    x = x.to(dtype)
    _check(x, "nvfp4", g)
    _check(x, "nvfp4", torch.tensor(g, device="cuda"))
    _check(x, "nvfp4", torch.tensor([g], device="cuda", dtype=BF16))
    _check(x, "nvfp4", torch.tensor(g, device="cuda", dtype=F16))
    _check(x, "mxfp4")


def test_every_half_against_every_border():
    """All finite fp16 values over scales whose borders they meet; blocks of one value and its block's largest."""
    bits = torch.arange(0x7C00, dtype=torch.int16, device="cuda").view(F16)
    for lead in (6.0, 1.0, 448.0, 0.0625, 65504.0):
        x = torch.full((bits.numel(), 16), lead, device="cuda", dtype=F16)
        x[:, 3] = torch.minimum(bits, torch.full_like(bits, lead))
        x[:, 4] = -x[:, 3]
        for g in (1.0, 2.0 ** -7, 0.1):
            _check(x, "nvfp4", g)
        _check(x, "mxfp4")


@pytest.mark.parametrize("g", [2.0 ** -140, 2.0 ** -126, 1e-30, 3e-20, 1e15, 1e25, 2.0 ** 100, 3e38])
def test_scales_over_the_whole_range(g):
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(40, 128, device="cuda", generator=gen).double() * g * 100
    x *= torch.exp2(torch.randint(-12, 6, (40, 8, 1), device="cuda", generator=gen).double()).expand(40, 8, 16).reshape(40, 128)
    x = x.clamp(-3.3e38, 3.3e38).float()
    x[0, :16] = 0
    x[1, :16] = 1e38   # saturates under the small ones
    x[2, :16] = 1e-40  # and vanishes under the large ones
    t = quantize_fp4(x, scale=torch.tensor(g, device="cuda"))
    code, byte, _ = _reference(x.double().cpu().numpy(), "nvfp4", float(np.float32(g)))
    got_code, got_byte = _unpack(t)
    assert (got_byte == byte).all() and (got_code == code).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("g", [2.0 ** -12, 2.0 ** -60, 2.0 ** -140, 0.001, 1e-25, 1e-42, 1.0, 2.0 ** 20])
def test_the_types_largest_values_keep_their_sign(dtype, g):
    """Quotients beyond fp32's range saturate to 6 with the value's sign."""
    big = torch.finfo(dtype).max
    gen = torch.Generator(device="cuda").manual_seed(31)
    x = torch.randn(8, 64, device="cuda", generator=gen)
    x[0, 5], x[1, 17], x[2, 40:44] = -big, big, -big
    x[3, :16] = torch.where(torch.arange(16, device="cuda") % 2 == 0, big, -big)
    x = x.to(dtype)
    t = quantize_fp4(x, scale=torch.tensor(g, device="cuda"))
    code, byte, _ = _reference(x.double().cpu().numpy(), "nvfp4", float(np.float32(g)))
    got_code, got_byte = _unpack(t)
    assert (got_byte == byte).all() and (got_code == code).all(), np.argwhere(got_code != code)[:5]
    _check(x, "mxfp4")
    _check(x, "nvfp4")


def test_power_of_two_scales_over_the_whole_range():
    e = torch.arange(-149, 128, device="cuda")
    x = torch.ldexp(torch.ones(277, device="cuda", dtype=torch.float64), e)[:, None]
    x = (x * (1 + torch.arange(32, device="cuda") / 32.0)).clamp(max=3.4e38).float()
    t = quantize_fp4(x, format="mxfp4")
    code, byte, _ = _reference(x.double().cpu().numpy(), "mxfp4", 1.0)
    got_code, got_byte = _unpack(t)
    assert (got_byte[:, :1] == byte).all() and (got_code == code).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_zeros_infinities_and_nan(fmt, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(140, 100, device="cuda", generator=gen).to(dtype)
    x[3] = 0
    x[5, 40:60] = 0
    x[7, 33] = float("nan")
    x[130, 99] = float("inf")
    x[131, 0] = -float("inf")
    _check(x, fmt, 0.01 if fmt == "nvfp4" else None)
    if fmt == "nvfp4":  # the tensor's own scale: everything is NaN, and says so
        assert dequantize_fp4(quantize_fp4(x)).isnan().all()
        for bad in (float("nan"), float("inf"), -1.0):
            _check(x, fmt, torch.tensor(bad, device="cuda"))
        zero = torch.zeros(3, 40, device="cuda", dtype=dtype)
        assert (dequantize_fp4(_check(zero, fmt)) == 0).all()
        assert (dequantize_fp4(quantize_fp4(torch.ones_like(zero), scale=torch.zeros((), device="cuda"))) == 0).all()


def _nearest_on_device(t, grid):
    """_nearest on the device: the same comparisons of 64-bit quotients."""
    grid = torch.from_numpy(grid).to(t.device)
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.bucketize(t, mid), torch.bucketize(t, mid, right=True)
    return torch.where(lo % 2 == 0, lo, hi)


def _check_on_device(x, fmt, given):
    """What _check does for finite matrices, without leaving the device (many values)."""
    t = quantize_fp4(x, format=fmt, scale=given)
    rows, cols = x.shape
    block = BLOCK[fmt]
    v = torch.nn.functional.pad(x.double(), (0, -cols % block)).view(rows, -1, block)
    most = v.abs().amax(-1)
    if fmt == "nvfp4":
        g = (x.double().abs().max() / 2688).float() if given is None else torch.tensor(given, dtype=F32, device="cuda")
        assert torch.equal(t.scale, g)
        byte = _nearest_on_device(most / (6 * g.double()), E4M3)
        unit = torch.from_numpy(E4M3).cuda()[byte] * g.double()
    else:
        byte = torch.where(most > 0, torch.frexp(most)[1] - 3 + 127, 0).clamp(0, 254)
        unit = torch.ldexp(torch.ones_like(most), byte - 127)
    quotient = torch.where(unit[..., None] > 0, v.abs() / torch.where(unit > 0, unit, 1)[..., None], 0)
    code = _nearest_on_device(quotient, E2M1)
    want = torch.copysign(torch.from_numpy(E2M1).cuda()[code] * unit[..., None], v).view(rows, -1)[:, :cols]
    code = torch.where(unit[..., None] > 0, code | torch.signbit(v).long() << 3, 0).view(rows, -1)[:, :cols]
    got = torch.stack([t.values & 15, t.values >> 4], -1).view(rows, -1)
    assert torch.equal(got[:, :cols].long(), code) and not got[:, cols:].any()
    got = t.scales.permute(0, 3, 2, 1, 4).reshape(-1, t.scales.shape[1] * 4)[:rows]
    assert torch.equal(got[:, :byte.shape[1]].long(), byte.long()) and not got[:, byte.shape[1]:].any()
    for dtype in (F32, BF16, F16):
        assert torch.equal(dequantize_fp4(t, dtype), want.float().to(dtype))


@pytest.mark.parametrize("fmt,own", [("nvfp4", True), ("nvfp4", False), ("mxfp4", False)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [2731, 2720])
def test_more_runs_than_threads(cols, dtype, fmt, own):
    """4001 rows of 86 runs of 32 values, padding included, are more than the
    303104 threads of the quantiser and twice the 151552 of its amax pass, and
    no whole number of rounds; rows on 16 bytes and off them."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(4001, cols, device="cuda", generator=gen) * torch.exp(torch.randn(4001, 1, device="cuda", generator=gen))
    x = x.clamp(-60, 60)
    for run in (100, 200000, 310000, 344083) if own else (None,):
        y = x.clone()
        if run is not None:  # the largest lies in a thread's first, second and third run, and near the last one
            per_row = (cols + 63) // 64 * 2
            y[run // per_row, min(run % per_row * 32 + 5, cols - 1)] = -77.0
        _check_on_device(y.to(dtype), fmt, None if fmt == "mxfp4" or own else 0.0173)


@pytest.mark.parametrize("scale_dtype", [BF16, F16, F32])
def test_a_scale_of_minus_zero_is_zero(scale_dtype):
    x = torch.ones(3, 40, device="cuda")
    t = _check(x, "nvfp4", torch.tensor(-0.0, device="cuda", dtype=scale_dtype))
    assert (dequantize_fp4(t) == 0).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_alignment_and_leading_dimensions(fmt, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(4, 37, 200, device="cuda", generator=gen).to(dtype)
    _check(base[:, :, 1:98], fmt)             # off 16 bytes, strided rows
    _check(base[1, :, :96], fmt)              # strided rows on 16 bytes
    _check(base[:, 2:30, :64], fmt)           # leading dimensions that do not fold
    _check(base[0, 0], fmt)                   # one dimension
    _check(base[0, :1].expand(9, 200), fmt)   # expanded rows
    _check(base.transpose(0, 1)[:, :, :32], fmt)
    _check(base[:, :, :1], fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_empty_and_out(fmt):
    e = quantize_fp4(torch.empty(0, 48, device="cuda"), format=fmt)
    assert e.rows == 0 and dequantize_fp4(e).shape == (0, 48)
    if fmt == "nvfp4":
        assert float(e.scale) == 0
        assert float(quantize_fp4(torch.empty(2, 0, 48, device="cuda"), scale=0.5).scale) == 0.5
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 70, 90, device="cuda", generator=gen).bfloat16()
    want = quantize_fp4(x, format=fmt)
    out = quantize_fp4(torch.zeros_like(x), format=fmt)
    got = quantize_fp4(x, format=fmt, out=out)
    assert got is out and torch.equal(dequantize_fp4(out), dequantize_fp4(want))
    buf = torch.empty(2, 70, 90, device="cuda", dtype=F16)
    assert dequantize_fp4(out, F16, out=buf) is buf
    assert torch.equal(buf, dequantize_fp4(want, F16))


def test_shared_scale_of_the_ranks():
    """The scale that shard.SharedActivationScale gives goes in as it is."""
    from dgx_monarch_b200.shard import SharedActivationScale

    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(3, 50, 256, device="cuda", generator=gen).bfloat16()
    shared = SharedActivationScale()
    try:
        scale = shared(x)
        assert scale.dtype == BF16
        _check(x, "nvfp4", scale)
    finally:
        shared.close()


def test_streams_and_graphs():
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(500, 640, device="cuda", generator=gen).bfloat16()
    want = dequantize_fp4(quantize_fp4(x))
    torch.cuda.synchronize()
    outs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [dequantize_fp4(quantize_fp4(x)) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            back = dequantize_fp4(quantize_fp4(x))
        graphs.append((graph, back))
    x.copy_(3 * torch.randn(500, 640, device="cuda", generator=gen))
    for graph, _ in graphs:
        graph.replay()
    want = dequantize_fp4(quantize_fp4(x))
    torch.cuda.synchronize()
    assert all(torch.equal(back, want) for _, back in graphs)

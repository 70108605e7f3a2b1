"""The product of two microscaled 4-bit tensors against 64 bits.

Exact cases: integer codes and scales of small powers of two make every
partial sum a multiple of 2^-4 below 2^19, which fp32 holds exactly in any
order, so the result has to be equal.

Tolerance of the others.  Products of two codes are multiples of 1/4 up to 36
and a block's 16 of them sum exactly (12 bits), times two scales (8 bits): 20
bits, exact in fp32.  What rounds are the additions of the blocks' sums, at
most ceil(k / 16) + 8 (for a split K) of them, each off by at most a step of
the running sum, 2^-23 of S = sum |terms|; then three fp32 operations (the two
tensor scales and the bias, 2^-24 each of the result's terms) and the rounding
to the output's type, eps / 2.
"""
from __future__ import annotations

import pytest
import torch

from dgx_monarch_b200.fp4 import Fp4Tensor, dequantize_fp4, fp4_matmul, quantize_fp4
from dgx_monarch_b200.fp4 import scales_shape, values_shape

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _random(g, rows, cols, fmt, dtype=BF16):
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    t = quantize_fp4(x.to(dtype), format=fmt)
    used = torch.zeros(t.scales.shape[0] * 128, dtype=torch.bool, device="cuda")
    used[:rows] = True  # bytes of rows past the last are nobody's: NaN there must not show
    t.scales[~used.view(-1, 4, 32)[:, None].expand(-1, t.scales.shape[1], -1, -1).transpose(2, 3)] = 0xFF
    return t


def _exact_values(t):
    unit = t if t.scale is None else Fp4Tensor(t.values, t.scales, t.shape, t.format, torch.ones_like(t.scale))
    v = dequantize_fp4(unit, F32).double()  # code * s: exact
    return v.reshape(-1, t.cols) * (1.0 if t.scale is None else float(t.scale))


def _check(a, b, bias=None, out_dtype=BF16, out=None):
    got = fp4_matmul(a, b, bias=bias, out_dtype=out_dtype, out=out)
    x, w = _exact_values(a), _exact_values(b)
    want, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    tol = ((a.cols + 15) // 16 + 8) * 2.0 ** -23 * size + 3 * 2.0 ** -24 * size \
        + torch.finfo(out_dtype).eps / 2 * 1.001 * want.abs() + torch.finfo(out_dtype).tiny
    assert got.shape == (*a.shape[:-1], b.rows) and got.dtype == out_dtype
    off = (got.reshape(-1, b.rows).double() - want).abs() / tol
    assert torch.isfinite(got).all() and float(off.max()) <= 1, (float(off.max()), off.argmax())
    return got


SIZES = [(1, 1, 1), (1, 8, 16), (2, 256, 64), (16, 130, 100), (17, 300, 96), (33, 129, 257), (64, 640, 512),
         (65, 129, 320), (128, 256, 1024), (300, 77, 1000), (1000, 50, 320), (700, 20, 65), (500, 9, 2000),
         (129, 1280, 5120), (257, 511, 127), (5, 5120, 2049), (1003, 777, 1000), (2560, 2304, 288), (3000, 4001, 33),
         (4, 1000, 3000), (20, 900, 3000), (50, 600, 3000), (2300, 2700, 700), (2301, 2699, 700), (1100, 3100, 2000),
         (1030, 3001, 2100), (3, 5000, 5120), (30, 3300, 5120), (10, 1900, 3600), (5000, 7, 2600), (2800, 64, 4000),
         # narrow tiles, K split 2 .. 8 ways; 192 columns; CTA pairs, rows on and off 16 bytes
         (5, 1900, 1700), (300, 100, 3000), (400, 200, 3500)]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_exact_sums(fmt, m, n, k):
    """Every code and scale byte in its place, whatever the tile, the split and the tails."""
    g = _gen(m + 3 * n + 7 * k)

    def tensor(rows):
        values = torch.zeros(values_shape(rows, k), device="cuda", dtype=torch.uint8)
        code = torch.randint(0, 16, (rows, 2 * values.shape[1]), device="cuda", generator=g, dtype=torch.uint8)
        code[:, k:] = 0
        values[:] = code[:, 0::2] | code[:, 1::2] << 4
        shape = scales_shape(rows, k, fmt)
        e = torch.randint(-1, 2, shape, device="cuda", generator=g)
        byte = ((e + 7) << 3 if fmt == "nvfp4" else e + 127).to(torch.uint8)
        block = 16 if fmt == "nvfp4" else 32
        blocks = torch.arange(shape[1], device="cuda")[:, None, None, None] * 4 + torch.arange(4, device="cuda")
        byte[:, (blocks * block >= k).expand(shape[1:])] = 0
        return Fp4Tensor(values, byte, (rows, k), fmt, torch.ones((), device="cuda") if fmt == "nvfp4" else None)

    a, b = tensor(m), tensor(n)
    got = fp4_matmul(a, b, out_dtype=F32)
    want = _exact_values(a) @ _exact_values(b).T
    assert torch.equal(got.double(), want), ((got - want).abs().max(), (got.double() != want).sum())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 700, 500), (3, 257, 5120), (40, 1000, 272), (200, 136, 768), (1500, 1000, 400),
                                   (2300, 2600, 640), (1100, 3100, 2000)])
def test_random_tensors_with_bias(fmt, out_dtype, m, n, k):
    g = _gen(m + n)
    a, b = _random(g, m, k, fmt), _random(g, n, k, fmt)
    bias = torch.randn(n, device="cuda", generator=g)
    first = _check(a, b, bias.to(out_dtype), out_dtype)
    _check(a, b, bias, out_dtype)
    _check(a, b, None, out_dtype)
    assert torch.equal(first, fp4_matmul(a, b, bias=bias.to(out_dtype), out_dtype=out_dtype))


@pytest.mark.parametrize("m", [1, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257])
def test_every_row_count_around_a_tile(m):
    g = _gen(m)
    _check(_random(g, m, 208, "nvfp4"), _random(g, 384, 208, "nvfp4"), None, F32)
    _check(_random(g, 384, 208, "mxfp4"), _random(g, m, 208, "mxfp4"), None, F32)


def test_leading_dimensions_outputs_and_empty():
    g = _gen(1)
    x = torch.randn(3, 7, 96, device="cuda", generator=g).bfloat16()
    a, b = quantize_fp4(x), _random(g, 40, 96, "nvfp4")
    want = _check(a, b)
    assert want.shape == (3, 7, 40)
    wide = torch.full((3, 7, 60), 7.0, device="cuda", dtype=BF16)
    got = fp4_matmul(a, b, out=wide[:, :, 3:43])   # rows of 60, a base off 16 bytes
    assert torch.equal(got, want) and (wide[:, :, :3] == 7).all() and (wide[:, :, 43:] == 7).all()
    one = quantize_fp4(x[0, 0])
    assert fp4_matmul(one, b).shape == (40,)
    empty = quantize_fp4(torch.empty(0, 96, device="cuda"))
    assert fp4_matmul(empty, b).shape == (0, 40) and fp4_matmul(b, empty).shape == (40, 0)


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n", [(1, 57), (300, 57), (2475, 57), (2048, 513), (1024, 2041), (600, 1001), (2301, 2699)])
def test_columns_behind_the_output_stay(m, n, out_dtype):
    """Aligned output rows that end inside 16 bytes."""
    g = _gen(m + n)
    a, b = _random(g, m, 320, "nvfp4"), _random(g, n, 320, "nvfp4")
    want = _check(a, b, None, out_dtype)
    wide = torch.full((m + 1, (n + 15) // 8 * 8), 7.0, device="cuda", dtype=out_dtype)
    assert torch.equal(fp4_matmul(a, b, out_dtype=out_dtype, out=wide[:m, :n]), want)
    assert (wide[:, n:] == 7).all() and (wide[m:] == 7).all()


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,pad,first", [(300, 57, 0, 0), (40, 193, 5, 2), (2475, 300, 3, 1), (1024, 2041, 0, 0),
                                           (2301, 2699, 2, 1), (500, 2048, 8, 3)])
def test_output_rows_off_16_bytes(m, n, pad, first, out_dtype):
    g = _gen(m * n)
    a, b = _random(g, m, 320, "nvfp4"), _random(g, n, 320, "nvfp4")
    want = _check(a, b, None, out_dtype)
    wide = torch.full((m + 1, n + pad), 7.0, device="cuda", dtype=out_dtype).flatten()
    out = wide[first:first + m * (n + pad)].view(m, n + pad)[:, :n]  # odd bases, strides, or both
    assert torch.equal(fp4_matmul(a, b, out_dtype=out_dtype, out=out), want)
    rest = torch.ones_like(wide, dtype=torch.bool)
    rest[first:first + m * (n + pad)].view(m, n + pad)[:, :n] = False
    assert (wide[rest] == 7).all()


# More tiles than CTAs (or CTA pairs) at one time: 320 and 256 tiles on 74 pairs, in the first with rows on 16 bytes
# whatever the type; 157 and 313 of 16, 32 and 64 columns on 148 CTAs, either operand's rows as the tile's; 216 of 192.
MANY_TILES = [(4000, 5000, 2000), (4000, 4097, 1500), (9, 20000, 300), (20000, 9, 300), (30, 20001, 300),
              (20000, 30, 300), (50, 40000, 300), (20000, 60, 300), (3000, 1600, 2100)]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", MANY_TILES)
def test_many_tiles_exact_sums(fmt, m, n, k):
    test_exact_sums(fmt, m, n, k)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(4000, 5000, 2000), (4000, 4097, 1500), (9, 20000, 300), (20000, 30, 300),
                                   (3000, 1600, 2100)])
def test_many_tiles_with_bias(fmt, out_dtype, m, n, k):
    """_check's bound, for sums that may also leave a 16-bit type: the border
    between its largest value and infinity is half a step above that value
    (fp16: 65504 + 16).  A sum above it by more than the fp32 error has to be
    infinite, with its sign, and none below it by more may be."""
    g = _gen(m + n)
    a, b = _random(g, m, k, fmt), _random(g, n, k, fmt)
    bias = torch.randn(n, device="cuda", generator=g)
    got = fp4_matmul(a, b, bias=bias, out_dtype=out_dtype)
    x, w = _exact_values(a), _exact_values(b)
    want, size = x @ w.T + bias.double(), x.abs() @ w.abs().T + bias.double().abs()
    info = torch.finfo(out_dtype)
    fp32_error = ((k + 15) // 16 + 8) * 2.0 ** -23 * size + 3 * 2.0 ** -24 * size
    border = info.max * (1 + info.eps / 2 / (2 - info.eps))  # max = (2 - eps) 2^e, half its step = eps / 2 2^e
    over = got.isinf()
    assert not got.isnan().any()
    assert (want.abs() + fp32_error >= border)[over].all() and (got[over].double().sign() == want[over].sign()).all()
    assert not (want.abs() - fp32_error > border)[~over].any()
    tol = fp32_error + info.eps / 2 * 1.001 * want.abs() + info.tiny
    assert ((got.double() - want).abs() <= tol)[~over].all()
    assert torch.equal(got, fp4_matmul(a, b, bias=bias, out_dtype=out_dtype))


@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_many_tiles_leave_the_rest_of_the_output(out_dtype):
    """CTA pairs with several tiles each, rows on 16 bytes in a wider matrix: nothing before, behind or below is touched."""
    g = _gen(11)
    m, n = 4000, 4100
    a, b = _random(g, m, 600, "nvfp4"), _random(g, n, 600, "nvfp4")
    want = _check(a, b, None, out_dtype)
    wide = torch.full((m + 1, n + 44), 7.0, device="cuda", dtype=out_dtype)
    assert torch.equal(fp4_matmul(a, b, out_dtype=out_dtype, out=wide[:m, 16:16 + n]), want)
    assert (wide[:, :16] == 7).all() and (wide[:, 16 + n:] == 7).all() and (wide[m] == 7).all()


def test_one_plan_on_another_alignment_and_from_two_threads():
    """Sizes and strides of the output alike, bases on 16 bytes and off them; and threads that call at the same time."""
    import threading

    g = _gen(12)
    a, b = _random(g, 90, 512, "nvfp4"), _random(g, 256, 512, "nvfp4")
    x = torch.randn(90 * 512 + 8, device="cuda", generator=g).bfloat16()
    want = _check(a, b)
    flat = torch.empty(90 * 256 + 8, device="cuda", dtype=BF16)
    for first in (0, 1, 8, 5):
        assert torch.equal(fp4_matmul(a, b, out=flat[first:first + 90 * 256].view(90, 256)), want)
    chains = {}
    for first in (0, 1, 8, 5):
        rows = x[first:first + 90 * 512].view(90, 512)
        chains[first] = rows, fp4_matmul(quantize_fp4(rows), b), fp4_matmul(quantize_fp4(rows, scale=0.01), b)
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(first):
        try:
            rows = chains[first][0]
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                got[first] = [(fp4_matmul(quantize_fp4(rows), b), fp4_matmul(quantize_fp4(rows, scale=0.01), b))
                              for _ in range(50)]
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 - shown below, from the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(first,)) for first in chains]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for first, calls in got.items():
        assert all(torch.equal(u, chains[first][1]) and torch.equal(v, chains[first][2]) for u, v in calls)


def test_nan_scales_stay_in_their_row_and_column():
    g = _gen(2)
    x = torch.randn(200, 320, device="cuda", generator=g).bfloat16()
    w = torch.randn(130, 320, device="cuda", generator=g).bfloat16()
    for fmt, scale in (("nvfp4", 0.01), ("mxfp4", None)):
        want = fp4_matmul(quantize_fp4(x, format=fmt, scale=scale), quantize_fp4(w, format=fmt, scale=scale))
        y, v = x.clone(), w.clone()
        y[77, 200] = float("nan")
        v[5, 319] = float("inf")
        got = fp4_matmul(quantize_fp4(y, format=fmt, scale=scale), quantize_fp4(v, format=fmt, scale=scale))
        assert got[77].isnan().all() and got[:, 5].isnan().all()
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[77] = keep[:, 5] = False
        assert torch.equal(got[keep], want[keep])


def test_streams_graphs_and_two_calls_at_once():
    g = _gen(3)
    b = _random(g, 1536, 1024, "nvfp4")
    xs = [torch.randn(m, 1024, device="cuda", generator=g).bfloat16() for m in (2, 300, 2048)]
    want = [fp4_matmul(quantize_fp4(x), b) for x in xs]
    torch.cuda.synchronize()
    outs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [[fp4_matmul(quantize_fp4(x), b) for x in xs] for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for per in outs for o, w in zip(per, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [fp4_matmul(quantize_fp4(x), b) for x in xs]
        graphs.append((graph, got))
    for x in xs:
        x.copy_(torch.randn_like(x))
    for graph, _ in graphs:
        graph.replay()
    want = [fp4_matmul(quantize_fp4(x), b) for x in xs]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for _, got in graphs for o, w in zip(got, want))


def test_block_of_a_transformer():
    """The operators as a block uses them: a 4-bit QKV projection, the heads'
    norm and rotation in place, attention, and a 4-bit output projection,
    against the same chain in 64 bits from the same packed tensors.

    The attention's own bound against 64 bits is 5e-3 relative (2-norm) in
    bf16; the projections and the norm add a bf16 rounding each (2^-8 at the
    most, 2^-9 in the 2-norm's mean) and requantisation moves a value by at
    most half a step of e2m1 (1/4 relative, in a few values at a border): the
    last product is therefore taken from the kernel's own packed tensor."""
    from dgx_monarch_b200.ops import attention_fwd
    from dgx_monarch_b200.prologue import rope_table
    from dgx_monarch_b200.qk_norm import qk_norm_rope

    g = _gen(4)
    rows, heads, hid = 320, 4, 512
    x = torch.randn(1, rows, hid, device="cuda", generator=g).bfloat16()
    w_qkv = quantize_fp4((torch.randn(3 * hid, hid, device="cuda", generator=g) * hid ** -0.5).bfloat16())
    w_out = quantize_fp4((torch.randn(hid, hid, device="cuda", generator=g) * hid ** -0.5).bfloat16())
    wq, wk = ((1 + 0.2 * torch.randn(128, device="cuda", generator=g)).bfloat16() for _ in range(2))
    pos = torch.stack([torch.arange(rows, device="cuda") // 20, torch.arange(rows, device="cuda") % 20], 1)
    rope = rope_table(pos, [64, 64])
    xq = quantize_fp4(x)
    qkv = fp4_matmul(xq, w_qkv).view(1, rows, 3, heads, 128)
    q, k, v = qkv.unbind(2)
    qk_norm_rope(q, k, norm_q_w=wq, norm_k_w=wk, rope=rope, q_out=q, k_out=k)
    attn, _ = attention_fwd(q, k, v)
    packed = quantize_fp4(attn.flatten(2))
    y = _check(packed, w_out)

    qkv64 = (_exact_values(xq) @ _exact_values(w_qkv).T).view(rows, 3, heads, 128)

    def side(t, w):
        n = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        c, s = rope.double()[:, None, :, 0], rope.double()[:, None, :, 1]
        a, b = n[..., 0::2], n[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2).transpose(0, 1)

    p = torch.softmax(side(qkv64[:, 0], wq) @ side(qkv64[:, 1], wk).transpose(1, 2) / 128 ** 0.5, -1)
    want = (p @ qkv64[:, 2].transpose(0, 1)).transpose(0, 1).reshape(rows, hid)
    rel = float((attn.flatten(2)[0].double() - want).norm() / want.norm())
    assert rel <= 5e-3 + 3 * 2.0 ** -8, rel
    assert y.shape == (1, rows, hid)

"""Refusals of the Linear calls, all before any device work."""
from __future__ import annotations

import ctypes
import shutil

import pytest
import torch

FAKE = 1 << 20  # aligned placeholder address, never dereferenced


@pytest.fixture(scope="module")
def lib():
    from dgx_monarch_b200 import _build, _lib

    if not _build.LIB_PATH.exists():
        if shutil.which("nvcc") is None:
            pytest.skip("libdgxm_sp.so is not built and nvcc is absent")
        _build.build_library()
    return _lib.load()


def _desc(**kw):
    from dgx_monarch_b200 import _lib

    d = _lib.LinearDesc()
    d.m, d.n, d.k = 4, 64, 128
    d.x_stride = d.w_stride = 128
    d.out_stride = d.residual_stride = d.pre_stride = 64
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def _forward(lib, d, x=FAKE, w=FAKE, bias=None, gate=None, residual=None, out=FAKE, pre=None, work=None, size=0):
    return lib.dgxm_linear(d, x, w, bias, gate, residual, out, pre, work, size, None)


def _backward(lib, d, grads, dout=FAKE, x=FAKE, w=FAKE, gate=None, pre=None, work=None, size=0):
    from dgx_monarch_b200 import _lib

    pointers = _lib.LinearGradPointers(**grads) if grads is not None else None
    return lib.dgxm_linear_backward(d, pointers, dout, x, w, gate, pre, work, size, None)


@pytest.mark.parametrize("kw,code,needle", [
    ({"m": -1}, 1, "product"),
    ({"k": 0}, 1, "product"),
    ({"m": 2 ** 30 + 1}, 1, "product"),
    ({"k": 2 ** 24 + 1, "x_stride": 2 ** 25, "w_stride": 2 ** 25}, 2, "2^24"),
    ({"n": 2 ** 24 + 8, "out_stride": 2 ** 25}, 2, "2^24"),
    ({"dtype": 3}, 2, "dtype 3"),
    ({"dtype": 2}, 2, "dtype 2"),
    ({"out_dtype": 1}, 2, "dtype 1"),
    ({"bias_dtype": 2}, 2, "dtype 2"),
    ({"activation": 4}, 2, "activation 4"),
    ({"gate_form": 5}, 1, "form 5"),
    ({"gate_form": 2, "sample_rows": 0}, 1, "whole samples"),
    ({"gate_form": 2, "sample_rows": 3}, 1, "whole samples"),
    ({"x_stride": 127}, 1, "below its row"),
    ({"w_stride": 0}, 1, "below its row"),
    ({"out_stride": 63}, 1, "below its row"),
    ({"m": 2 ** 30, "n": 2 ** 24, "out_stride": 2 ** 24}, 2, "tiles"),
])
def test_c_refusals(lib, kw, code, needle):
    d = _desc(**kw)
    assert _forward(lib, d) == code
    assert needle in lib.dgxm_last_error_message().decode()
    assert lib.dgxm_linear_workspace(d, FAKE, FAKE) == -1
    assert _backward(lib, d, {"x": FAKE}) == code


def test_empty_products(lib):
    assert _forward(lib, _desc(m=0), x=None, out=None) == 0
    assert _forward(lib, _desc(n=0), w=None, out=None) == 0
    assert _backward(lib, _desc(m=0), {"x": FAKE}, dout=None, x=None) == 0


@pytest.mark.parametrize("kw,args,needle", [
    ({}, {"x": None}, "NULL"),
    ({}, {"w": None}, "NULL"),
    ({}, {"out": None}, "NULL"),
    ({}, {"x": FAKE + 1}, "aligned"),
    ({}, {"out": FAKE + 1}, "aligned"),
    ({"bias_dtype": 3}, {"bias": FAKE + 2}, "aligned"),
    ({}, {"gate": FAKE}, "gate_form"),
    ({"gate_form": 1, "sample_rows": 4}, {}, "gate_form"),
    ({"residual_stride": 3}, {"residual": FAKE}, "below its row"),
    ({"pre_stride": 63}, {"pre": FAKE}, "below its row"),
    ({}, {"x": FAKE + 2}, "workspace"),
    ({"x_stride": 129}, {}, "workspace"),
    ({"w_stride": 129}, {"work": FAKE, "size": 64 * 128 * 2 - 1}, "workspace"),
])
def test_c_pointer_refusals(lib, kw, args, needle):
    assert _forward(lib, _desc(**kw), **args) == 1
    assert needle in lib.dgxm_last_error_message().decode()


@pytest.mark.parametrize("kw,grads,args,needle", [
    ({}, None, {}, "NULL gradients"),
    ({}, {"x": FAKE}, {"dout": None}, "upstream"),
    ({}, {"x": FAKE}, {"w": None}, "NULL operand"),
    ({}, {"w": FAKE}, {"x": None}, "NULL operand"),
    ({}, {"gate": FAKE}, {}, "gate"),
    ({"gate_form": 1, "sample_rows": 4}, {"x": FAKE}, {}, "gate"),
    ({"activation": 1}, {"x": FAKE}, {}, "without pre"),
    ({"gate_form": 1, "sample_rows": 4}, {"gate": FAKE}, {"gate": FAKE}, "without pre"),
    ({"activation": 1, "pre_stride": 3}, {"x": FAKE}, {"pre": FAKE}, "below its row"),
    ({}, {"x": FAKE + 1}, {}, "aligned"),
    ({"activation": 1}, {"x": FAKE}, {"pre": FAKE}, "workspace"),
    ({}, {"bias": FAKE}, {}, "workspace"),
    ({"out_dtype": 3}, {"x": FAKE}, {}, "workspace"),
])
def test_c_gradient_refusals(lib, kw, grads, args, needle):
    assert _backward(lib, _desc(**kw), grads, **args) == 1
    assert needle in lib.dgxm_last_error_message().decode()


def test_workspaces(lib):
    from dgx_monarch_b200 import _lib

    assert lib.dgxm_linear_workspace(_desc(), FAKE, FAKE) == 0
    assert lib.dgxm_linear_workspace(_desc(), FAKE + 8, FAKE) == 4 * 128 * 2
    assert lib.dgxm_linear_workspace(_desc(k=127), FAKE, FAKE) == 0  # rows on 16 bytes, whatever they hold
    assert lib.dgxm_linear_workspace(_desc(k=127, w_stride=127), FAKE, FAKE) == 64 * 128 * 2
    grads = _lib.LinearGradPointers(x=FAKE, w=FAKE)
    assert lib.dgxm_linear_backward_workspace(_desc(), grads, FAKE, FAKE, FAKE) == 0
    assert lib.dgxm_linear_backward_workspace(_desc(activation=1), grads, FAKE, FAKE, FAKE) == 4 * 64 * 2
    assert lib.dgxm_linear_backward_workspace(_desc(), None, FAKE, FAKE, FAKE) == -1


def test_python_refuses_host_tensors():
    from dgx_monarch_b200.linear import linear, linear_backward

    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_backward(torch.zeros(4, 8, dtype=torch.bfloat16), x, w)


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,error,needle", [
    ({"x": _t(64)}, ValueError, "x must be"),
    ({"x": _t(2, 4, 64, dtype=torch.float32)}, TypeError, "float32"),
    ({"w": _t(8, 63)}, ValueError, "matrix"),
    ({"w": _t(8, 64, dtype=torch.float16)}, TypeError, "share one dtype"),
    ({"bias": _t(9)}, ValueError, "bias"),
    ({"bias": _t(8, dtype=torch.float16)}, ValueError, "bias"),
    ({"bias": _t(8, 2)[:, 0]}, ValueError, "contiguous"),
    ({"activation": "relu"}, ValueError, "relu"),
    ({"gate": _t(8, dtype=torch.float16)}, TypeError, "gate"),
    ({"gate": _t(3, 8)}, ValueError, "gate"),
    ({"gate": _t(2, 4, 9)}, ValueError, "gate"),
    ({"x": _t(2, 4, 0), "w": _t(8, 0)}, ValueError, "no columns"),
])
def test_python_argument_checks(monkeypatch, args, error, needle):
    from dgx_monarch_b200 import linear

    monkeypatch.setattr(linear, "_require_cuda", lambda *a: None)
    call = {"x": _t(2, 4, 64), "w": _t(8, 64), "bias": None, "activation": "none", "gate": None, **args}
    with pytest.raises(error, match=needle):
        linear._describe(**call)


def test_gate_forms(monkeypatch):
    from dgx_monarch_b200 import _lib, linear

    monkeypatch.setattr(linear, "_require_cuda", lambda *a: None)
    form = lambda x, gate: (lambda d: (d.gate_form, d.sample_rows, tuple(d.gate_stride)))(
        linear._describe(x, _t(8, 64), None, "none", gate))
    x3, x2, one = _t(2, 4, 64), _t(6, 64), _t(3, 1, 64)
    assert form(x3, _t(8)) == (_lib.MOD_SHARED, 4, (0, 0))
    assert form(x3, _t(2, 8)) == form(x3, _t(2, 1, 8)) == (_lib.MOD_SAMPLE, 4, (8, 0))
    assert form(x3, _t(2, 4, 8)) == (_lib.MOD_TOKEN, 4, (32, 8))
    assert form(x2, _t(8))[0] == _lib.MOD_SHARED and form(x2, _t(6, 8)) == (_lib.MOD_TOKEN, 6, (48, 8))
    assert form(one, _t(3, 8)) == (_lib.MOD_TOKEN, 1, (8, 0))


def test_row_strides():
    from dgx_monarch_b200.linear import _row_stride

    assert _row_stride(_t(4, 64)) == 64 and _row_stride(_t(4, 96)[:, :64]) == 96
    assert _row_stride(_t(2, 4, 64)) == 64 and _row_stride(_t(2, 4, 96)[..., :64]) == 96
    assert _row_stride(_t(2, 8, 64)[:, :4]) is None and _row_stride(_t(1, 8, 64)[:, :4]) == 64
    assert _row_stride(_t(4, 2, 64).transpose(0, 1)) is None and _row_stride(_t(64, 4).T) is None
    assert _row_stride(_t(1, 64).expand(4, 64)) is None and _row_stride(_t(5, 1, 64)) == 64


def test_output_checks(monkeypatch, lib):
    from dgx_monarch_b200 import linear as ln

    monkeypatch.setattr(ln, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(ln, "launch", lambda *a: None)
    x, w = _t(2, 4, 64), _t(8, 64)
    with pytest.raises(ValueError, match="out"):
        ln.linear(x, w, out=_t(2, 4, 9))
    with pytest.raises(ValueError, match="rows of its own"):
        ln.linear(x, w, out=_t(2, 8, 8)[:, :4])
    with pytest.raises(ValueError, match="rows of its own"):
        ln.linear(x, w, out=_t(1, 1, 8).expand(2, 4, 8))
    with pytest.raises(TypeError, match="out_dtype"):
        ln.linear(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="residual"):
        ln.linear(x, w, residual=_t(2, 4, 8, dtype=torch.float32))
    with pytest.raises(ValueError, match="memory of x or w"):
        ln.linear(_t(8, 64), _t(64, 64), out=None) is None or ln.linear(x, _t(64, 64), out=x)
    with pytest.raises(ValueError, match="pre"):
        ln.linear_backward(_t(2, 4, 8), x, w, activation="silu")
    with pytest.raises(ValueError, match="dout"):
        ln.linear_backward(_t(2, 4, 9), x, w)
    out, pre = ln.linear(x, w, return_pre=True, out_dtype=torch.float32)
    assert out.dtype == torch.float32 and pre.dtype == x.dtype
    grads = ln.linear_backward(_t(2, 4, 8), x, w, w_grad=False, bias=_t(8, dtype=torch.float32))
    assert grads.w is None and grads.bias.dtype == torch.float32 and grads.x.shape == x.shape
    assert all(g is None for g in ln.linear_backward(_t(2, 4, 8), x, w, x_grad=False, w_grad=False))
    with pytest.raises(RuntimeError, match="no_grad"):
        ln.linear(x, w.float().requires_grad_(True).bfloat16())


def test_long_contractions_of_a_gradient(lib):
    """w's gradient is a product along m: as long as k may be, no longer; the other gradients take any m."""
    from dgx_monarch_b200 import _lib

    d = _desc(m=2 ** 24 + 64, n=8, out_stride=8, k=8, x_stride=8, w_stride=8)
    assert _backward(lib, d, {"w": FAKE}) == 2 and "2^24" in lib.dgxm_last_error_message().decode()
    need = lambda **g: lib.dgxm_linear_backward_workspace(d, _lib.LinearGradPointers(**g), FAKE, FAKE, FAKE)
    assert need(w=FAKE) == -1 and need(x=FAKE) >= 0 and need(bias=FAKE) > 0
    d.m = 2 ** 24
    assert need(w=FAKE) >= 0


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc is absent")
def test_struct_layouts(tmp_path):
    """Sizes and offsets of the new descriptors, as gcc lays out the header's."""
    import ctypes
    import subprocess
    from pathlib import Path

    from dgx_monarch_b200 import _lib

    header = Path(__file__).resolve().parents[1] / "include" / "dgxm_sp.h"
    structs = {"dgxm_block_norm_desc": _lib.BlockNormDesc, "dgxm_block_norm_grads": _lib.BlockNormGradPointers,
               "dgxm_linear_desc": _lib.LinearDesc, "dgxm_linear_grads": _lib.LinearGradPointers}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    source = tmp_path / "layout.c"
    source.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void) {{ {" ".join(lines)} return 0; }}\n')
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(source)], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert [int(v) for v in out.split()] == want


@pytest.mark.parametrize("x_shape,gate_shape", [((2, 0, 64), (8,)), ((2, 0, 64), (2, 8)), ((2, 0, 64), (2, 1, 8)),
                                                ((1, 0, 64), (1, 8)), ((0, 64), (1, 8)), ((0, 64), (8,)), ((2, 0, 64), (2, 0, 8)),
                                                ((0, 4, 64), (0, 8))])
def test_gradients_of_no_rows_are_zeros(monkeypatch, lib, x_shape, gate_shape):
    """A sum over no rows is zero, whatever the memory held and however many samples have no rows."""
    from dgx_monarch_b200 import linear as ln

    monkeypatch.setattr(ln, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(ln, "launch", lambda *a: None)
    monkeypatch.setattr(torch, "empty_like", lambda t, **kw: torch.full_like(t, float("nan")))
    x, w, bias, gate = _t(*x_shape), _t(8, 64), _t(8), _t(*gate_shape)
    dout = _t(*x_shape[:-1], 8)
    grads = ln.linear_backward(dout, x, w, bias=bias, gate=gate, pre=dout)
    for got, like in zip(grads, (x, w, bias, gate)):
        assert torch.equal(got, torch.zeros_like(like))


@pytest.mark.parametrize("form", ["shared", "token", "token apart"])
def test_partial_sums_of_many_short_samples(lib, form):
    """The workspace of a bias' gradient goes by the rows, not by the samples, where no sum is a sample's; one wanted sum
    takes half of two."""
    from dgx_monarch_b200 import _lib

    m, n = 9450, 13824
    need = lambda rows, **g: lib.dgxm_linear_backward_workspace(
        _desc(m=m, n=n, out_stride=n, pre_stride=n, gate_form=_lib.MOD_SHARED if form == "shared" else _lib.MOD_TOKEN, sample_rows=rows,
              gate_stride=(ctypes.c_int64 * 2)(*((0, 0) if form == "shared" else (2 * rows * n if form == "token apart" else rows * n, n)))),
        _lib.LinearGradPointers(**g), FAKE, FAKE, FAKE)
    whole = need(m, bias=FAKE)
    assert whole == -(-m // 64) * n * 4
    assert need(1, bias=FAKE) == whole  # (rows of samples of one are always a step apart)
    assert need(3, bias=FAKE) == (m // 3 * n * 4 if form == "token apart" else whole)
    assert need(1, bias=FAKE, gate=FAKE) == whole * (2 if form == "shared" else 1)

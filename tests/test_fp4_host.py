"""Refusals of the 4-bit calls, all before any device work, and the C structs
of the operators' descriptors."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

FAKE = 1 << 20  # aligned placeholder address, never dereferenced
HEADER = Path(__file__).resolve().parents[1] / "include" / "dgxm_sp.h"


@pytest.fixture(scope="module")
def lib():
    from dgx_monarch_b200 import _build, _lib

    if not _build.LIB_PATH.exists():
        if shutil.which("nvcc") is None:
            pytest.skip("libdgxm_sp.so is not built and nvcc is absent")
        _build.build_library()
    return _lib.load()


def _quant(**kw):
    from dgx_monarch_b200 import _lib

    d = _lib.Fp4Desc()
    d.rows, d.cols, d.row_stride, d.scale_dtype = 4, 64, 64, _lib.DTYPE_F32
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def _gemm(**kw):
    from dgx_monarch_b200 import _lib

    d = _lib.Fp4GemmDesc()
    d.m, d.n, d.k, d.out_stride = 4, 64, 64, 64
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def _message(lib, needle):
    assert needle in lib.dgxm_last_error_message().decode()


@pytest.mark.parametrize("kw,code,needle", [
    ({"format": 2}, 2, "format 2"),
    ({"rows": -1}, 1, "-1 x 64"),
    ({"cols": 0}, 1, "4 x 0"),
    ({"cols": 2 ** 31}, 1, "matrix"),
    ({"dtype": 2}, 2, "dtype 2"),
    ({"row_stride": 63}, 1, "row stride 63"),
    ({"scale_dtype": 2}, 2, "scale dtype 2"),
    ({"rows": 2 ** 31}, 2, "blocks"),
])
def test_quantisation_descriptors(lib, kw, code, needle):
    d = _quant(**kw)
    assert lib.dgxm_quantize_fp4(d, FAKE, FAKE, FAKE, FAKE, FAKE, None, 0, None) == code
    _message(lib, needle)
    if "scale_dtype" not in kw and kw.get("format", 0) == 0:
        assert lib.dgxm_dequantize_fp4(d, FAKE, FAKE, FAKE, FAKE, None) == code


def test_quantisation_arguments(lib):
    q = lib.dgxm_quantize_fp4
    assert q(None, FAKE, FAKE, FAKE, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(), None, FAKE, FAKE, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(), FAKE, FAKE, FAKE + 8, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(), FAKE + 1, FAKE, FAKE, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(), FAKE, FAKE + 2, FAKE, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(), FAKE, FAKE, FAKE, FAKE, None, None, 0, None) == 1
    _message(lib, "scale_out")
    assert q(_quant(), FAKE, None, FAKE, FAKE, FAKE, None, 0, None) == 1
    _message(lib, "workspace")
    need = lib.dgxm_quantize_fp4_workspace()
    assert q(_quant(), FAKE, None, FAKE, FAKE, FAKE, FAKE, need - 1, None) == 1
    assert q(_quant(scale_value=-1.0), FAKE, None, FAKE, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(scale_value=float("nan")), FAKE, None, FAKE, FAKE, FAKE, None, 0, None) == 1
    assert q(_quant(format=1), FAKE, FAKE, FAKE, FAKE, None, None, 0, None) == 1
    _message(lib, "mxfp4")
    assert q(_quant(format=1, rows=0), None, None, None, None, None, None, 0, None) == 0
    d = lib.dgxm_dequantize_fp4
    assert d(_quant(), FAKE, FAKE, None, FAKE, None) == 1
    assert d(_quant(format=1), FAKE, FAKE, FAKE, FAKE, None) == 1
    assert d(_quant(rows=0), None, None, FAKE, None, None) == 0


@pytest.mark.parametrize("kw,code,needle", [
    ({"format": 7}, 2, "format 7"),
    ({"m": -1}, 1, "product"),
    ({"k": 0}, 1, "product"),
    ({"n": 2 ** 31}, 1, "product"),
    ({"k": 2 ** 24 + 1}, 2, "k 16777217"),
    ({"out_dtype": 2}, 2, "dtype 2"),
    ({"bias_dtype": 9}, 2, "dtype 9"),
    ({"out_stride": 63}, 1, "row stride 63"),
    ({"m": 2 ** 30, "n": 2 ** 30, "out_stride": 2 ** 30}, 2, "tiles"),
    ({"m": 0}, 0, ""),
    ({"n": 0}, 0, ""),
])
def test_product_descriptors(lib, kw, code, needle):
    rc = lib.dgxm_fp4_matmul(_gemm(**kw), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, None)
    assert rc == code
    if code:
        _message(lib, needle)


def test_product_arguments(lib):
    ok = [FAKE] * 6 + [None, FAKE]

    def call(at, value, d=None):
        args = list(ok)
        args[at] = value
        return lib.dgxm_fp4_matmul(d or _gemm(), *args, None)

    assert lib.dgxm_fp4_matmul(None, *ok, None) == 1
    for at in (0, 1, 3, 4, 7):
        assert call(at, None) == 1
    for at in (0, 1, 3, 4):
        assert call(at, FAKE + 8) == 1
    for at in (2, 5):
        assert call(at, None) == 1
        _message(lib, "scales")
        assert call(at, FAKE + 2) == 1
    assert call(6, FAKE + 1) == 1 and call(7, FAKE + 1) == 1
    assert call(0, FAKE, _gemm(format=1)) == 1


def test_packed_sizes(lib):
    from dgx_monarch_b200.fp4 import scales_shape, values_shape

    for rows, cols in ((0, 1), (1, 1), (127, 31), (128, 32), (129, 65), (3, 1000)):
        assert lib.dgxm_fp4_values_bytes(rows, cols) == torch.Size(values_shape(rows, cols)).numel()
        for code, fmt in enumerate(("nvfp4", "mxfp4")):
            assert lib.dgxm_fp4_scales_bytes(rows, cols, code) == torch.Size(scales_shape(rows, cols, fmt)).numel()
    assert lib.dgxm_fp4_values_bytes(1, 0) == -1 and lib.dgxm_fp4_scales_bytes(1, 1, 5) == -1


def _packed(rows=4, cols=64, fmt="nvfp4", **kw):
    from dgx_monarch_b200.fp4 import Fp4Tensor, scales_shape, values_shape

    args = {"values": torch.zeros(values_shape(rows, cols), dtype=torch.uint8),
            "scales": torch.zeros(scales_shape(rows, cols, fmt), dtype=torch.uint8), "shape": (rows, cols),
            "format": fmt, "scale": torch.ones(()) if fmt == "nvfp4" else None}
    args.update(kw)
    return Fp4Tensor(**args)


def test_packed_tensor_checks():
    assert _packed().rows == 4 and _packed(fmt="mxfp4").scale is None
    assert _packed(6, 64, shape=(2, 3, 64)).rows == 6
    for kw in ({"values": torch.zeros(4, 31, dtype=torch.uint8)}, {"values": torch.zeros(4, 32)},
               {"scales": torch.zeros(1, 2, 32, 4, 4, dtype=torch.uint8)}, {"shape": (4, 0)}, {"shape": ()},
               {"shape": (5, 64)}, {"format": "fp4"}, {"scale": None}, {"scale": torch.ones(2)},
               {"scale": torch.ones((), dtype=torch.bfloat16)}):
        with pytest.raises(ValueError):
            _packed(**kw)


def test_python_refuses_host_tensors():
    from dgx_monarch_b200.fp4 import dequantize_fp4, fp4_matmul, quantize_fp4

    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_fp4(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        dequantize_fp4(_packed())
    with pytest.raises(RuntimeError, match="CUDA"):
        fp4_matmul(_packed(), _packed())


@pytest.mark.parametrize("make,error", [
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), format="int4"), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64, dtype=torch.float64)), TypeError),
    (lambda f: f.quantize_fp4(torch.zeros(())), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 0)), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(64, 4).t()), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), format="mxfp4", scale=1.0), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), scale=0.0), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), scale=1e-50), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), scale=float("inf")), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), scale=torch.ones(2)), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), scale=torch.ones((), dtype=torch.float64)), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), out=_packed(5, 64)), ValueError),
    (lambda f: f.quantize_fp4(torch.zeros(4, 64), out=_packed(fmt="mxfp4")), ValueError),
    (lambda f: f.dequantize_fp4(_packed(), torch.float64), TypeError),
    (lambda f: f.dequantize_fp4(_packed(), torch.float32, out=torch.zeros(4, 63)), ValueError),
    (lambda f: f.dequantize_fp4(_packed(), torch.float32, out=torch.zeros(2, 2, 64)), ValueError),
    (lambda f: f.dequantize_fp4(_packed(), torch.float32, out=torch.zeros(64, 4).t()), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(fmt="mxfp4")), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(cols=65)), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(), out_dtype=torch.float64), TypeError),
    (lambda f: f.fp4_matmul(_packed(), _packed(), bias=torch.zeros(5)), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(), bias=torch.zeros(8)[::2]), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(), out=torch.zeros(4, 4)), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(), out=torch.zeros(4, 4, dtype=torch.bfloat16).t()), ValueError),
    (lambda f: f.fp4_matmul(_packed(), _packed(), out=torch.zeros(1, 4, dtype=torch.bfloat16).expand(4, 4)), ValueError),
])
def test_python_argument_checks(monkeypatch, make, error):
    """Sizes and types, on host tensors with the device check off; none of these calls reaches the library."""
    from dgx_monarch_b200 import fp4

    monkeypatch.setattr(fp4, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(fp4, "launch", lambda *a: pytest.fail("launched"))
    with pytest.raises(error):
        make(fp4)


def test_a_number_as_scale_is_no_part_of_the_plan(monkeypatch):
    """Scales that change from call to call make one plan, and drop no other operator's; each call gets its own."""
    from dgx_monarch_b200 import _call, fp4

    got = []
    monkeypatch.setattr(_call, "_PLANS", {"another operator's": object()})
    monkeypatch.setattr(fp4, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(fp4, "launch", lambda name, index, desc, *a: got.append(desc))
    x = torch.zeros(4, 64)
    scales = [1.0 + i / 1024 for i in range(2 * _call._MOST_PLANS)]
    for scale in scales:
        fp4.quantize_fp4(x, scale=scale)
    assert len(_call._PLANS) == 2 and "another operator's" in _call._PLANS
    assert [d.scale_value for d in got] == scales  # exact in fp32
    for bad in (0.0, -1.0, 1e-50, float("inf"), float("nan"), 1e39):  # with the plan there
        with pytest.raises(ValueError, match="scale"):
            fp4.quantize_fp4(x, scale=bad)
    fp4.quantize_fp4(x, scale=torch.ones(()))
    assert got[-1].scale_value == 0.0 and len(got) == len(scales) + 1


def test_no_autograd_graph():
    from dgx_monarch_b200 import _call

    w = torch.zeros(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        _call.no_graph("", w)
    with torch.no_grad():
        _call.no_graph("", w)


def test_every_tensor_that_requires_a_gradient_is_refused(monkeypatch):
    """The scale of a packed tensor and an output to write into among them."""
    from dgx_monarch_b200 import fp4, qk_norm

    for module in (fp4, qk_norm):
        monkeypatch.setattr(module, "_require_cuda", lambda *a: None)
        monkeypatch.setattr(module, "launch", lambda *a: None)
    x, bias = torch.zeros(4, 64), torch.zeros(4)
    learned = _packed(scale=torch.ones((), requires_grad=True))
    out, out_q = torch.zeros(4, 4, requires_grad=True), torch.zeros(1, 4, 2, 64, requires_grad=True)
    q = torch.zeros(1, 4, 2, 64)
    made = fp4.quantize_fp4(x)
    made.scale.requires_grad_(True)
    calls = [lambda: fp4.quantize_fp4(x, out=learned), lambda: fp4.dequantize_fp4(learned),
             lambda: fp4.dequantize_fp4(made),
             lambda: fp4.dequantize_fp4(_packed(), torch.float32, out=torch.zeros(4, 64, requires_grad=True)),
             lambda: fp4.fp4_matmul(learned, _packed()), lambda: fp4.fp4_matmul(_packed(), learned),
             lambda: fp4.fp4_matmul(_packed(), _packed(), out_dtype=torch.float32, out=out),
             lambda: fp4.fp4_matmul(_packed(), _packed(), bias=bias.clone().requires_grad_()),
             lambda: qk_norm.qk_norm_rope(q, q.clone(), q_out=out_q),
             lambda: qk_norm.qk_norm_rope(q, q.clone(), k_out=out_q)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc is absent")
def test_struct_layouts_match_the_header(tmp_path):
    from dgx_monarch_b200 import _lib

    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    want = {}
    for cls, name in ((_lib.QkNormDesc, "dgxm_qk_norm_desc"), (_lib.Fp4Desc, "dgxm_fp4_desc"),
                      (_lib.Fp4GemmDesc, "dgxm_fp4_gemm_desc")):
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        want[name] = ctypes.sizeof(cls)
        for field, _ in cls._fields_:
            lines.append(f'  printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
            want[f"{name}.{field}"] = getattr(cls, field).offset
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert {k: int(v) for k, v in (line.rsplit(" ", 1) for line in out.splitlines())} == want

"""Refusals of the block norm calls, all before any device work, and the
64-bit gradient formulas of the tests against differences."""
from __future__ import annotations

import shutil

import pytest
import torch

from tests import block_reference as ref

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

    d = _lib.BlockNormDesc()
    d.batch, d.seq, d.width, d.norm_mode = 1, 4, 64, _lib.BLOCK_NORM_LAYER
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def _forward(lib, d, x=FAKE, branch=None, gate=None, scale=None, shift=None, norm_w=None, norm_b=None, branch_w=None,
             x_out=None, out=FAKE):
    return lib.dgxm_block_norm(d, x, branch, gate, scale, shift, norm_w, norm_b, branch_w, x_out, out, None)


def _backward(lib, d, grads, dy=FAKE, dx_out=FAKE, x_out=FAKE, branch=None, gate=None, scale=None, norm_w=None, norm_b=None,
              branch_w=None, work=None, size=0):
    from dgx_monarch_b200 import _lib

    pointers = _lib.BlockNormGradPointers(**grads) if grads is not None else None
    return lib.dgxm_block_norm_backward(d, pointers, dy, dx_out, x_out, branch, gate, scale, norm_w, norm_b, branch_w, work,
                                        size, None)


@pytest.mark.parametrize("kw,code,needle", [
    ({"batch": -1}, 1, "negative"),
    ({"seq": -1}, 1, "negative"),
    ({"width": 0}, 2, "width 0"),
    ({"width": 8193}, 2, "width 8193"),
    ({"dtype": 2}, 2, "dtype 2"),
    ({"weight_dtype": 1}, 2, "dtype 1"),
    ({"mod_dtype": 1}, 2, "dtype 1"),
    ({"norm_mode": 3}, 2, "norm mode 3"),
    ({"gate_form": 4}, 1, "form 4"),
    ({"mod_form": -1}, 1, "form -1"),
    ({"eps": -1.0}, 1, "eps"),
    ({"eps": float("nan")}, 1, "eps"),
    ({"seq": 0}, 0, ""),
    ({"batch": 0}, 0, ""),
])
def test_c_refusals(lib, kw, code, needle):
    d = _desc(**kw)
    assert _forward(lib, d) == code
    if code:
        assert needle in lib.dgxm_last_error_message().decode()
        assert lib.dgxm_block_norm_backward_workspace(d) == -1
    assert _backward(lib, d, {"x": FAKE}) == code


@pytest.mark.parametrize("kw,args,needle", [
    ({}, {"x": None}, "NULL x"),
    ({}, {"x": FAKE + 1}, "aligned"),
    ({}, {"out": None}, "out"),
    ({}, {"branch": FAKE}, "x_out"),
    ({}, {"x_out": FAKE}, "x_out"),
    ({"norm_mode": 0}, {"out": None}, "neither"),
    ({"norm_mode": 0}, {"branch": FAKE, "x_out": FAKE}, "out"),
    ({"norm_mode": 0, "mod_form": 2}, {"branch": FAKE, "x_out": FAKE, "out": None, "scale": FAKE}, "without a norm"),
    ({"norm_mode": 0}, {"branch": FAKE, "x_out": FAKE, "out": None, "norm_w": FAKE}, "without a norm"),
    ({"gate_form": 2}, {"gate": FAKE}, "without a branch"),
    ({"branch_norm": 1}, {}, "without a branch"),
    ({}, {"branch": FAKE, "x_out": FAKE, "branch_w": FAKE}, "branch_w"),
    ({"norm_mode": 2}, {"norm_b": FAKE}, "norm_b"),
    ({}, {"branch": FAKE, "x_out": FAKE, "gate": FAKE}, "gate_form"),
    ({"gate_form": 1}, {"branch": FAKE, "x_out": FAKE}, "gate_form"),
    ({}, {"scale": FAKE}, "mod_form"),
    ({"mod_form": 3}, {}, "mod_form"),
    ({"mod_form": 3}, {"shift": FAKE + 1}, "aligned"),
    ({}, {"norm_w": FAKE + 1}, "aligned"),
])
def test_c_pointer_refusals(lib, kw, args, needle):
    assert _forward(lib, _desc(**kw), **args) == 1
    assert needle in lib.dgxm_last_error_message().decode()


@pytest.mark.parametrize("kw,grads,args,needle", [
    ({}, None, {}, "NULL gradients"),
    ({}, {}, {}, "gradient of x"),
    ({}, {"x": FAKE}, {"dy": None}, "upstream"),
    ({}, {"x": FAKE}, {"x_out": None}, "upstream"),
    ({"norm_mode": 0}, {}, {"dx_out": None}, "neither"),
    ({}, {"x": FAKE, "branch": FAKE}, {}, "without a branch"),
    ({}, {"x": FAKE, "branch": FAKE}, {"branch": FAKE}, "pass NULL"),
    ({}, {"x": FAKE, "gate": FAKE}, {"branch": FAKE}, "gate"),
    ({"gate_form": 2}, {"x": FAKE}, {"branch": FAKE}, "gate"),
    ({}, {"x": FAKE, "scale": FAKE}, {}, "mod_form"),
    ({"mod_form": 2}, {"x": FAKE, "scale": FAKE}, {}, "without the scale"),
    ({}, {"x": FAKE, "branch_w": FAKE}, {"branch": FAKE}, "branch_w"),
    ({"norm_mode": 2}, {"x": FAKE, "norm_b": FAKE}, {}, "norm_b"),
    ({"norm_mode": 0}, {"norm_w": FAKE}, {}, "without a norm"),
    ({}, {"x": FAKE, "norm_w": FAKE}, {}, "workspace"),
    ({}, {"x": FAKE + 1}, {}, "aligned"),
])
def test_c_gradient_refusals(lib, kw, grads, args, needle):
    assert _backward(lib, _desc(**kw), grads, **args) == 1
    assert needle in lib.dgxm_last_error_message().decode()


def test_workspace(lib):
    d = _desc(seq=4096)
    need = lib.dgxm_block_norm_backward_workspace(d)
    assert need >= 3 * 64 * 4
    assert _backward(lib, d, {"x": FAKE, "norm_w": FAKE}, work=FAKE, size=need - 1) == 1
    assert lib.dgxm_block_norm_backward_workspace(_desc(seq=0)) == 0
    assert lib.dgxm_block_norm_backward_workspace(None) == -1


def test_python_refuses_host_tensors():
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    x = torch.zeros(1, 4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        block_norm(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        block_norm_backward(x, x, x)


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,error,needle", [
    ({"x": _t(4, 64)}, ValueError, "3-D"),
    ({"x": _t(2, 4, 64, dtype=torch.float64)}, TypeError, "float64"),
    ({"x": _t(2, 64, 4).transpose(1, 2)}, ValueError, "contiguous"),
    ({"branch": _t(2, 5, 64)}, ValueError, "branch"),
    ({"branch": _t(2, 4, 64, dtype=torch.float32)}, ValueError, "branch"),
    ({"gate": _t(64)}, ValueError, "without a branch"),
    ({"branch_norm": True}, ValueError, "without a branch"),
    ({"branch": _t(2, 4, 64), "branch_w": _t(64)}, ValueError, "without branch_norm"),
    ({"norm_mode": 7}, ValueError, "norm_mode 7"),
    ({"norm_mode": 0}, ValueError, "nothing to do"),
    ({"norm_mode": 0, "branch": _t(2, 4, 64), "scale": _t(64)}, ValueError, "NORM_NONE"),
    ({"norm_mode": 2, "norm_b": _t(64)}, ValueError, "NORM_LAYER"),
    ({"norm_w": _t(32)}, ValueError, "norm_w"),
    ({"norm_w": _t(64, dtype=torch.float16)}, ValueError, "norm_w"),
    ({"norm_w": _t(64), "norm_b": _t(64, dtype=torch.float32)}, TypeError, "share one dtype"),
    ({"scale": _t(3, 64)}, ValueError, "scale"),
    ({"scale": _t(2, 5, 64)}, ValueError, "scale"),
    ({"scale": _t(1, 4, 64)}, ValueError, "scale"),
    ({"scale": _t(2, 64), "shift": _t(64)}, ValueError, "both"),
    ({"scale": _t(2, 64), "shift": _t(2, 64, dtype=torch.float32)}, TypeError, "share one dtype"),
    ({"scale": _t(2, 64, dtype=torch.float16)}, TypeError, "scale"),
    ({"scale": _t(64, 2).T}, ValueError, "contiguous"),
])
def test_python_argument_checks(monkeypatch, args, error, needle):
    from dgx_monarch_b200 import block_norm

    monkeypatch.setattr(block_norm, "_require_cuda", lambda *a: None)
    call = {"x": _t(2, 4, 64), "branch": None, "gate": None, "branch_norm": False, "branch_w": None, "norm_mode": 1,
            "norm_w": None, "norm_b": None, "scale": None, "shift": None, "eps": 1e-6, **args}
    with pytest.raises(error, match=needle):
        block_norm._describe(**call)


def test_output_checks(monkeypatch, lib):
    from dgx_monarch_b200 import block_norm as bn

    monkeypatch.setattr(bn, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(bn, "launch", lambda *a: None)
    x, branch = _t(2, 4, 64), _t(2, 4, 64)
    with pytest.raises(ValueError, match="without a branch"):
        bn.block_norm(x, x_out=x)
    with pytest.raises(ValueError, match="NORM_NONE"):
        bn.block_norm(x, branch, norm_mode=bn.NORM_NONE, out=x)
    with pytest.raises(ValueError, match="share their memory"):
        bn.block_norm(x, branch, x_out=x, out=x)
    with pytest.raises(ValueError, match="other strides"):
        bn.block_norm(x[:, :, :32], out=x.view(-1)[:256].view(2, 4, 32))
    with pytest.raises(ValueError, match="expanded"):
        bn.block_norm(x, out=_t(1, 1, 64).expand(2, 4, 64))
    with pytest.raises(ValueError, match="contiguous"):
        bn.block_norm(x, out=_t(2, 64, 4).transpose(1, 2))
    with pytest.raises(ValueError, match="dy comes with a norm"):
        bn.block_norm_backward(None, x, x)
    with pytest.raises(ValueError, match="neither"):
        bn.block_norm_backward(None, None, x, branch, norm_mode=bn.NORM_NONE)
    with pytest.raises(ValueError, match="dy"):
        bn.block_norm_backward(_t(2, 4, 32), None, x)
    w = torch.zeros(64, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        bn.block_norm(torch.zeros(2, 4, 64), norm_w=w)
    with torch.no_grad():
        bn.block_norm(torch.zeros(2, 4, 64), norm_w=w)


def test_results_that_are_one_tensor(monkeypatch, lib):
    """Without a norm the stream's gradient is the upstream one; without a gate the branch's is the stream's."""
    from dgx_monarch_b200 import block_norm as bn

    monkeypatch.setattr(bn, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(bn, "launch", lambda *a: None)
    x, branch = _t(2, 4, 64), _t(2, 4, 64)
    assert bn.block_norm(x)[0] is x
    assert bn.block_norm(x, branch, norm_mode=bn.NORM_NONE)[1] is None
    up = _t(2, 4, 64)
    got = bn.block_norm_backward(None, up, x, branch, norm_mode=bn.NORM_NONE)
    assert got.x is up and got.branch is up
    got = bn.block_norm_backward(up, None, x, branch)
    assert got.branch is got.x and got.x.shape == x.shape
    got = bn.block_norm_backward(up, None, x, branch, gate=_t(1, 1, 64))
    assert got.branch is not got.x and got.gate.shape == (1, 1, 64) and got.scale is None


def test_upstream_gradients_of_any_strides(monkeypatch, lib):
    from dgx_monarch_b200 import block_norm as bn

    seen = []
    monkeypatch.setattr(bn, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(bn, "launch", lambda name, index, desc, out, dy, dx_out, *a: seen.append(
        (tuple(desc.dy_stride), tuple(desc.dx_out_stride), dy, dx_out)))
    x = _t(2, 4, 64)
    up, wide = torch.ones((), dtype=x.dtype).expand(2, 4, 64), _t(2, 4, 128)
    bn.block_norm_backward(up, wide[..., :64], x)
    assert seen[0][:2] == ((256, 64), (512, 128)) and seen[0][2] != up.data_ptr() and seen[0][3] == wide.data_ptr()


def test_numbers_held_in_tensors_are_read_in_each_call(monkeypatch, lib):
    from dgx_monarch_b200 import block_norm as bn

    seen = []
    monkeypatch.setattr(bn, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(bn, "launch", lambda name, index, desc, *a: seen.append(desc.eps))
    x, eps = _t(2, 4, 64), torch.tensor(0.25)
    for _ in range(2):
        bn.block_norm(x, eps=eps)
        bn.block_norm_backward(x, x, x, eps=eps)
        eps.fill_(0.5)
    assert seen == [0.25, 0.25, 0.5, 0.5]


@pytest.mark.parametrize("mode", ["layer", "rms", "none"])
@pytest.mark.parametrize("form", ["shared", "sample", "token"])
@pytest.mark.parametrize("branch_norm", [False, True])
def test_reference_gradients_against_differences(mode, form, branch_norm):
    """The tests' formulas in 64 bits: central differences of step h leave h^2 of the third derivative."""
    g = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    b, l, c = 2, 3, 7
    shape = {"shared": (c,), "sample": (b, c), "token": (b, l, c)}[form]
    args = {"x": rand(b, l, c), "branch": rand(b, l, c), "gate": rand(*shape),
            "branch_w": rand(c) if branch_norm else None}
    if mode != "none":
        args |= {"norm_w": rand(c), "norm_b": rand(c) if mode == "layer" else None, "scale": rand(*shape), "shift": rand(*shape)}
    dy, dr = (None if mode == "none" else rand(b, l, c)), rand(b, l, c)

    def loss(a):
        r, y, _, _ = ref.forward(**a, mode=mode, branch_norm=branch_norm)
        return (r * dr).sum() + (0 if y is None else (y * dy).sum())

    r = ref.forward(**args, mode=mode, branch_norm=branch_norm)[0]
    rest = {n: v for n, v in args.items() if n not in ("x", "branch")}
    grads = ref.backward(dy, dr, r, args["branch"], **rest, mode=mode, branch_norm=branch_norm)
    h = 1e-5
    for name, value in args.items():
        if value is None:
            continue
        way = rand(*value.shape)
        diff = (loss({**args, name: value + h * way}) - loss({**args, name: value - h * way})) / (2 * h)
        want = (grads[name][0] * way).sum()
        assert abs(diff - want) <= 1e-6 * (1 + (grads[name][0] * way).abs().sum()), name

"""Refusals of the Q/K norm + rotation calls, all before any device work: the
C entries with placeholder pointers, and the Python checks."""
from __future__ import annotations

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

    d = _lib.QkNormDesc()
    d.batch, d.seq, d.q_heads, d.k_heads, d.head_dim, d.rot_dim, d.norm_mode = 1, 4, 2, 2, 128, 128, _lib.NORM_HEAD
    for name, value in kw.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("kw,code,needle", [
    ({"batch": -1}, 1, "negative"),
    ({"head_dim": 0}, 2, "head_dim 0"),
    ({"head_dim": 100}, 2, "head_dim 100"),
    ({"head_dim": 264}, 2, "head_dim 264"),
    ({"rot_dim": 7}, 1, "rot_dim 7"),
    ({"rot_dim": 130}, 1, "rot_dim 130"),
    ({"dtype": 2}, 2, "dtype 2"),
    ({"weight_dtype": 1}, 2, "weight dtype 1"),
    ({"norm_mode": 1}, 2, "norm mode 1"),
    ({"eps": -1.0}, 1, "eps"),
    ({"eps": float("nan")}, 1, "eps"),
    ({"seq": 2 ** 31 - 1, "batch": 2}, 2, "head groups"),
    ({"seq": 2 ** 31 - 1, "batch": 2 ** 31 - 1}, 2, "head groups"),
    ({"seq": 2 ** 30}, 2, "head groups"),
    ({"q_heads": 2 ** 20 + 1}, 2, "heads"),
    ({"seq": 0}, 0, ""),
    ({"batch": 0}, 0, ""),
    ({"q_heads": 0, "k_heads": 0}, 0, ""),
])
def test_c_refusals(lib, kw, code, needle):
    d = _desc(**kw)
    assert lib.dgxm_qk_norm_rope(d, FAKE, FAKE, None, None, None, FAKE, FAKE, None) == code
    if code:
        assert needle in lib.dgxm_last_error_message().decode()
    rc = lib.dgxm_qk_norm_rope_backward(d, FAKE, FAKE, FAKE, FAKE, None, None, None, FAKE, FAKE, None, None, None, 0,
                                        None)
    assert rc == code


def test_c_pointer_refusals(lib):
    d = _desc()
    assert lib.dgxm_qk_norm_rope(None, FAKE, FAKE, None, None, None, FAKE, FAKE, None) == 1
    assert lib.dgxm_qk_norm_rope(d, None, FAKE, None, None, None, FAKE, FAKE, None) == 1
    assert lib.dgxm_qk_norm_rope(d, FAKE, FAKE, None, None, None, FAKE, None, None) == 1
    assert lib.dgxm_qk_norm_rope(d, FAKE + 1, FAKE, None, None, None, FAKE, FAKE, None) == 1
    assert lib.dgxm_qk_norm_rope(d, FAKE, FAKE, FAKE + 1, None, None, FAKE, FAKE, None) == 1
    assert lib.dgxm_qk_norm_rope(d, FAKE, FAKE, None, None, FAKE + 2, FAKE, FAKE, None) == 1
    # a call too large for one cluster: its weight gradients need the workspace
    d = _desc(seq=4096)
    args = [FAKE] * 4 + [FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE]
    assert lib.dgxm_qk_norm_rope_backward(d, *args, None, 0, None) == 1
    assert "workspace" in lib.dgxm_last_error_message().decode()
    need = lib.dgxm_qk_norm_rope_backward_workspace(d)
    assert lib.dgxm_qk_norm_rope_backward(d, *args, FAKE, need - 1, None) == 1
    assert lib.dgxm_qk_norm_rope_backward(d, None, *args[1:], FAKE, need, None) == 1
    assert lib.dgxm_qk_norm_rope_backward_workspace(_desc()) == 0
    assert lib.dgxm_qk_norm_rope_backward_workspace(_desc(q_heads=0, k_heads=0)) == 0
    assert lib.dgxm_qk_norm_rope_backward_workspace(_desc(seq=0)) == 0
    assert lib.dgxm_qk_norm_rope_backward_workspace(None) == -1
    assert lib.dgxm_qk_norm_rope_backward_workspace(_desc(head_dim=9)) == -1


def test_python_refuses_host_tensors():
    from dgx_monarch_b200.qk_norm import qk_norm_rope, qk_norm_rope_backward

    q = torch.zeros(1, 4, 2, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        qk_norm_rope(q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        qk_norm_rope_backward(q, q, q, q)


@pytest.mark.parametrize("change,error,needle", [
    ({"q": (4, 2, 128)}, ValueError, "4-D"),
    ({"k": (1, 5, 2, 128)}, ValueError, "does not share"),
    ({"k_dtype": torch.float16}, TypeError, "share one dtype"),
    ({"dtype": torch.float64}, TypeError, "float64"),
    ({"wq": (64,)}, ValueError, "norm_q_w"),
    ({"wq": (128,), "wk": None}, ValueError, "both norm weights"),
    ({"wq": (128,), "wk": (128,), "mode": 0}, ValueError, "NORM_NONE"),
    ({"rope": (3, 64, 2)}, ValueError, "rope"),
    ({"rope": (4, 65, 2)}, ValueError, "65 pairs"),
    ({"rope": (2, 4, 64, 2)}, ValueError, "rope"),
])
def test_python_argument_checks(monkeypatch, change, error, needle):
    """The checks of shapes and types, on host tensors with the device check off."""
    from dgx_monarch_b200 import qk_norm

    monkeypatch.setattr(qk_norm, "_require_cuda", lambda *a: None)
    dtype = change.get("dtype", torch.bfloat16)
    q = torch.zeros(change.get("q", (1, 4, 2, 128)), dtype=dtype)
    k = torch.zeros(change.get("k", (1, 4, 2, 128)), dtype=change.get("k_dtype", dtype))
    wq = torch.zeros(change["wq"], dtype=dtype) if change.get("wq") else None
    wk = torch.zeros(change["wk"], dtype=dtype) if change.get("wk") else wq if "wk" not in change else None
    rope = torch.zeros(change["rope"]) if "rope" in change else None
    with pytest.raises(error, match=needle):
        qk_norm._describe(q, k, change.get("mode", 2), wq, wk, 1e-6, rope, False)


def test_output_and_gradient_checks():
    from dgx_monarch_b200 import qk_norm

    like = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="q_out"):
        qk_norm._check_out("q_out", torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16), like)
    with pytest.raises(ValueError, match="q_out"):
        qk_norm._check_out("q_out", torch.zeros(1, 4, 2, 64), like)
    with pytest.raises(ValueError, match="expanded"):
        qk_norm._check_out("q_out", torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16).expand(1, 4, 2, 64), like)
    q, k = torch.zeros(1, 4, 2, 64), torch.zeros(1, 4, 2, 64)
    qk_norm._check_in_place("q_out", q, q, k)
    with pytest.raises(ValueError, match="other strides"):
        qk_norm._check_in_place("q_out", q.transpose(1, 2).reshape(1, 2, 4, 64)[:, :, :2], q[:, :2], k)
    with pytest.raises(ValueError, match="other tensor"):
        qk_norm._check_in_place("q_out", k, q, k)
    w = torch.zeros(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        qk_norm.no_graph("", None, w)
    with torch.no_grad():
        qk_norm.no_graph("", None, w)


@pytest.mark.parametrize("layout", ["expanded", "head_dim first", "head_dim of a wider step"])
def test_upstream_gradients_of_any_strides(lib, monkeypatch, layout):
    """One that a sum passes back, and others without a contiguous head_dim, reach the kernel as whole tensors."""
    from dgx_monarch_b200 import qk_norm

    seen = []

    def launch(name, index, desc, dq, dk, *rest):
        seen.append((tuple(desc.dq_stride), tuple(desc.dk_stride), dq, dk))

    monkeypatch.setattr(qk_norm, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(qk_norm, "launch", launch)

    def upstream(heads):
        if layout == "expanded":
            return torch.ones(()).expand(2, 3, heads, 64)
        if layout == "head_dim first":
            return torch.zeros(64, 2, 3, heads).permute(1, 2, 3, 0)
        return torch.zeros(2, 3, heads, 128)[..., ::2]

    q, k = torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 2, 64)
    dq, dk = upstream(4), upstream(2)
    gq, gk, _, _ = qk_norm.qk_norm_rope_backward(dq, dk, q, k)
    assert gq.shape == q.shape and gk.shape == k.shape
    (qs, ks, pq, pk), = seen
    assert qs == (3 * 4 * 64, 4 * 64, 64) and ks == (3 * 2 * 64, 2 * 64, 64)
    assert pq != dq.data_ptr() and pk != dk.data_ptr()
    qk_norm.qk_norm_rope_backward(q, k, q, k)  # whole ones as they are
    assert seen[1][2:] == (q.data_ptr(), k.data_ptr())
    with pytest.raises(ValueError, match="4-D"):
        qk_norm.qk_norm_rope_backward(torch.ones(()), dk, q, k)
    with pytest.raises(ValueError, match="contiguous head_dim"):
        qk_norm.qk_norm_rope_backward(q, k, q, dk)


def test_numbers_held_in_tensors_are_read_in_each_call(lib, monkeypatch):
    """An eps and an order of pairs that change in place between calls."""
    from dgx_monarch_b200 import qk_norm

    seen = []
    monkeypatch.setattr(qk_norm, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(qk_norm, "launch", lambda name, index, desc, *a: seen.append((desc.eps, desc.rope_halves)))
    q, rope = torch.zeros(1, 4, 2, 64), torch.zeros(4, 32, 2)
    eps, halves = torch.tensor(0.25), torch.tensor(False)
    for _ in range(2):
        qk_norm.qk_norm_rope(q, q.clone(), eps=eps, rope=rope, rope_halves=halves)
        qk_norm.qk_norm_rope_backward(q, q, q, q, eps=eps, rope=rope, rope_halves=halves)
        eps.fill_(0.5)
        halves.fill_(True)
    assert seen == [(0.25, 0), (0.25, 0), (0.5, 1), (0.5, 1)]

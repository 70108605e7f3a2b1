"""What every local operator refuses before a launch, on the host."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from dgx_monarch_b200._call import no_graph


def test_reverse_mode_is_refused():
    leaf = torch.zeros(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad.*here"):
        no_graph(" here", None, leaf)
    with torch.no_grad():
        no_graph("", None, leaf)
    no_graph("", torch.zeros(2), None)


def test_forward_mode_tangents_are_refused():
    """A dual tensor's tangent would be dropped: the outputs would be constants to the derivative."""
    x, w = torch.zeros(2), torch.zeros(2)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(2))
        with pytest.raises(RuntimeError, match="tangent"):
            no_graph("", w, None, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):  # which leaves forward mode on
            no_graph("", dual)
        no_graph("", w, x, forward_ad.unpack_dual(dual).primal)
    no_graph("", dual)


def test_operators_refuse_tangents(monkeypatch):
    from dgx_monarch_b200 import block_norm as bn
    from dgx_monarch_b200 import linear as ln

    monkeypatch.setattr(ln, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(bn, "_require_cuda", lambda *a: None)
    for module in (ln, bn):
        monkeypatch.setattr(module, "launch", lambda *a: pytest.fail("launched"))
    x, w = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="tangent"):
            ln.linear(dual, w)
        with pytest.raises(RuntimeError, match="tangent"):
            bn.block_norm(x, dual)

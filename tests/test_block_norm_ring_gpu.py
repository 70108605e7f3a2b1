"""Rows through the block norm's ring in shared memory: many to a slot, at every
offset to the 16-byte borders, every call's results looked at."""
from __future__ import annotations

import pytest
import torch

from tests.test_block_norm_gpu import TYPES, make, run_backward, run_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [333, 1001, 2731, 5119])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_slots_that_hold_rows_of_every_offset(width, kind):
    """Several rows a slot.  A row's ends are stored value by value where the next one's whole words land."""
    a, up = make(width, 2, max(2000, 5_000_000 // width), width, TYPES[kind], post=width < 2000)
    run_forward(a, "layer")
    run_backward(a, up, "layer")


@pytest.mark.parametrize("width,rows", [(5120, 4000), (2048, 6000), (8192, 2000), (1365, 4000), (515, 12000)])
def test_every_call_of_many(width, rows):
    """Sixty calls behind one another, the next one's blocks starting as the last one's end: all of them give the same bits."""
    from dgx_monarch_b200.block_norm import block_norm, block_norm_backward

    a, up = make(8, 1, rows, width, torch.bfloat16)
    rest = {n: t for n, t in a.items() if n != "x"}
    call = lambda: (*block_norm(**a), *(g for g in block_norm_backward(up["dy"], up["dr"], a["x"], **rest) if g is not None))
    want = call()
    differs = torch.zeros((), dtype=torch.bool, device="cuda")
    for _ in range(60):
        for got, first in zip(call(), want):
            differs |= (got != first).any()
    assert not differs


@pytest.mark.parametrize("width", [64, 77, 5120, 8191])
@pytest.mark.parametrize("rows", [1, 2, 3, 147, 149, 700, 1200])
def test_blocks_that_end_in_every_slot(width, rows):
    """Blocks whose rows fill no slot, some, all of them, and wrap around."""
    a, up = make(rows, 1, rows, width, torch.bfloat16)
    run_forward(a, "layer")
    run_backward(a, up, "layer")

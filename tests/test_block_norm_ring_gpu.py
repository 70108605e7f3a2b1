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

"""The in-tree build's options, on the CPU."""
from __future__ import annotations

import pytest


def test_tuning_defines_accept_only_the_kernel_macros(monkeypatch):
    from dgx_monarch_b200 import _build

    monkeypatch.setenv("DGXM_NVCC_DEFINES", "-DDGXM_SM_POLY_MOD=4 -DDGXM_SM_THR_BF16=6.0f")
    assert _build.tuning_defines() == ["-DDGXM_SM_POLY_MOD=4", "-DDGXM_SM_THR_BF16=6.0f"]
    monkeypatch.setenv("DGXM_NVCC_DEFINES", "-O0")
    with pytest.raises(ValueError, match="DGXM_"):
        _build.tuning_defines()
    monkeypatch.delenv("DGXM_NVCC_DEFINES")
    assert _build.tuning_defines() == []


def test_one_source_gives_one_library():
    """nvcc's own split compilation cuts the optimiser's work by what the threads happen to do: registers and spills of most
    kernels, and times by up to 40 %, went one way or the other from build to build."""
    from dgx_monarch_b200 import _build

    assert not any(f.startswith(("--split-compile", "-split-compile=")) and _build.NVCC_FLAGS[i - 1] != "-Xptxas"
                   for i, f in enumerate(_build.NVCC_FLAGS))


def test_every_source_is_part_of_one_unit():
    """A unit, or included by exactly one; kernels that report to the error word have their unit's."""
    import re

    from dgx_monarch_b200 import _build

    included = {u: re.findall(r'^#include "(\w+\.cu)"', (_build.CSRC / u).read_text(), re.M) for u in _build.UNITS}
    parts = sorted(_build.UNITS + [p for part in included.values() for p in part])
    assert parts == sorted(p.name for p in _build.CSRC.glob("*.cu"))
    for path in list(_build.CSRC.glob("*.cu")) + list(_build.CSRC.glob("*.cuh")):
        if path.name != "device_error.cuh":
            assert "__device__ int g_device_error" not in path.read_text()

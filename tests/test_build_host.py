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

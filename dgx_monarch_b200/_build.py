"""Build libdgxm_sp.so in-tree with nvcc for sm_100a.

The library's translation units are compiled side by side and linked against
the static CUDA runtime, so it loads next to any torch build without a JIT
cache.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_NAME = "libdgxm_sp.so"
LIB_PATH = PKG_DIR / LIB_NAME

UNITS = ["block_norm_bf16.cu", "block_norm_f16.cu", "block_norm_f32.cu", "dgxm_sp.cu", "linear.cu",
         "block_norm.cu"]  # the others are parts of dgxm_sp.cu

# ptxas takes a unit's kernels in parallel, which changes none.  nvcc's own
# --split-compile would cut the optimiser's work differently from run to run:
# two libraries of one source, one with 140-byte spills where the other has
# none, 61 us where the other takes 44.
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    *ARCH, "-lineinfo", "-O3", "-std=c++17",
    "-Xptxas", "-split-compile=0", "-Xcompiler", "-fPIC",
]
LINK_FLAGS = [*ARCH, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static"]


def _nvcc() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    cand = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    raise RuntimeError("nvcc was not found; set CUDA_HOME or put nvcc on PATH")


def _run(cmd: list[str]) -> str:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    return proc.stdout + proc.stderr


def sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h"))
                  + list((PKG_DIR.parent / "include").glob("*.h")))


def needs_build() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    return any(src.stat().st_mtime > built for src in sources())


def tuning_defines() -> list[str]:
    """Compile-time tuning of the kernels' defaults (the DGXM_SM_* macros of
    csrc/attn_fwd.cu), from DGXM_NVCC_DEFINES, e.g. "-DDGXM_SM_POLY_MOD=4".
    Only -D definitions are taken."""
    defines = os.environ.get("DGXM_NVCC_DEFINES", "").split()
    bad = [d for d in defines if not d.startswith("-DDGXM_")]
    if bad:
        raise ValueError(f"DGXM_NVCC_DEFINES takes -DDGXM_* definitions only, got {bad}")
    return defines


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile csrc/ into dgx_monarch_b200/libdgxm_sp.so.  A build with tuning
    defines is always redone, so the library matches them."""
    defines = tuning_defines()
    if not force and not defines and not needs_build():
        return LIB_PATH
    flags = NVCC_FLAGS + defines + (["-Xptxas", "-v"] if verbose else [])
    tmp = LIB_PATH.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as room, ThreadPoolExecutor(len(UNITS)) as side_by_side:
        objects = [str(Path(room) / unit) + ".o" for unit in UNITS]
        said = list(side_by_side.map(lambda unit, to: _run([_nvcc(), *flags, "-c", "-o", to, str(CSRC / unit)]), UNITS, objects))
        said.append(_run([_nvcc(), *LINK_FLAGS, "-o", str(tmp), *objects]))
    if verbose:
        print("".join(said))
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force=True, verbose=True))

"""Builds libb200kv.so (the C-ABI CUDA library) in-tree for sm_100a.

Usage: ``python -m torch_spyre_b200.build [--verbose]``.  The shared library is
written next to this file (``torch_spyre_b200/lib/libb200kv.so``) so it travels
with the source tree; nothing is installed.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

import torch

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "lib"
LIB_PATH = LIB_DIR / "libb200kv.so"


def fast_name() -> str:
    """File name of the Python module of csrc/fast_call.cpp: it fits one version of
    torch and of Python, so one built for another is not taken for it."""
    return f"_fast-{torch.__version__}-{sys.implementation.cache_tag}.so"


FAST_PATH = LIB_DIR / fast_name()
INCLUDE = PKG_DIR.parent / "include"

SOURCES = [
    "capi.cu",
    "kv_relayout.cu",
    "decode_attention.cu",
    "decode_mma.cu",
    "decode_simt.cu",
    "decode_noalloc.cu",
    "stick_relayout.cu",
    "fp8_ops.cu",
    "peer_allreduce.cu",
    "nvls_allreduce.cu",
    "rope.cu",
    "rotary.cu",
    "kv_rows.cu",
    "tree_attention.cu",
    "tree_mma_f16.cu",
    "tree_mma_bf16.cu",
    "lse_combine.cu",
    "oproj_allreduce.cu",
]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libb200kv")
    return cand


def _needs_rebuild() -> bool:
    if not LIB_PATH.exists():
        return True
    mtime = LIB_PATH.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return any(p.stat().st_mtime > mtime for p in deps)


def build_fast(force: bool = False) -> Path:
    """Compiles the module that calls the library without Python in between."""
    src = CSRC / "fast_call.cpp"
    if not force and FAST_PATH.exists() and FAST_PATH.stat().st_mtime >= src.stat().st_mtime:
        return FAST_PATH
    root = Path(torch.__file__).resolve().parent
    cuda_home = Path(nvcc_path()).resolve().parent.parent
    includes = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
                sysconfig.get_paths()["include"], cuda_home / "include"]
    tmp = FAST_PATH.with_name(FAST_PATH.name + ".tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{p}" for p in includes], str(src),
           "-o", str(tmp), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    try:
        proc = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"g++ could not be run: {e}") from e
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{' '.join(cmd)}\n{proc.stderr}")
    os.replace(tmp, FAST_PATH)
    return FAST_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles every CUDA source of the library into one shared object, and the
    module that calls it.  Only nvcc is needed: without the module (no g++, no
    Python headers) the same calls go through Python, which a warning says."""
    LIB_DIR.mkdir(exist_ok=True)
    if force or _needs_rebuild():
        _build_lib(verbose)
    try:
        build_fast(force)
    except RuntimeError as e:
        warnings.warn(f"the verification operators will be called through Python: {e}", RuntimeWarning, stacklevel=2)
    return LIB_PATH


def _build_lib(verbose: bool) -> None:
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [
        nvcc_path(),
        *ARCH_FLAGS,
        "-lineinfo",
        "-O3",
        "-t0",
        "-std=c++17",
        "--expt-relaxed-constexpr",
        "-Xcompiler",
        "-fPIC,-fvisibility=hidden",
        "-shared",
        f"-I{INCLUDE}",
        "-o",
        str(tmp),
        *[str(CSRC / s) for s in SOURCES],
    ]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{' '.join(cmd)}\n{proc.stderr}")
    if verbose:
        sys.stderr.write(proc.stderr)
    os.replace(tmp, LIB_PATH)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(LIB_PATH)

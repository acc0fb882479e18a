"""Build libhier_b200.so (all CUDA sources of the package) for sm_100a, and the
module that calls its small entry points from Python.

The library is built in-tree next to this file so that it travels with the
repository to the GPU machine.  ``python -m multics_b200.build`` rebuilds it;
``build(verbose=True)`` also prints ptxas register/shared-memory usage.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libhier_b200.so"
SOURCES = ["hier_capi.cu", "hier_meta.cu", "hier_prep.cu", "hier_attn.cu", "hier_selftest.cu",
           "hier_cached.cu", "hier_tiled.cu", "hier_shard.cu", "hier_bwd.cu", "hier_head_norm.cu",
           "hier_paged8.cu", "hier_paged8_attn.cu", "hier_paged8_mma.cu"]
BIND = PKG / "_bind.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def build_bind(force: bool = False) -> Path:
    """The Python module of csrc/bind.cpp (host code, PyTorch's headers)."""
    src = CSRC / "bind.cpp"
    deps = [src, CSRC / "pycall.h", ROOT / "include" / "hier_b200.h"]
    if BIND.exists() and not force:
        if BIND.stat().st_mtime >= max(d.stat().st_mtime for d in deps):
            return BIND
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    tmp = BIND.with_suffix(".so.tmp")
    includes = [ROOT / "include", sysconfig.get_paths()["include"], *include_paths("cuda")]
    libs = library_paths("cuda")
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{p}" for p in includes), "-o", str(tmp), str(src), *(f"-L{p}" for p in libs),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-lcudart"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"{cmd[0]} failed building {BIND.name}")
    os.replace(tmp, BIND)
    return BIND


def build(verbose: bool = False, force: bool = False) -> Path:
    build_bind(force)
    srcs = [CSRC / s for s in SOURCES if (CSRC / s).exists()]
    deps = srcs + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + [ROOT / "include" / "hier_b200.h"]
    if LIB.exists() and not force:
        newest = max(p.stat().st_mtime for p in deps)
        if LIB.stat().st_mtime >= newest:
            return LIB
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
           "-I", str(ROOT / "include"), "-o", str(tmp), *map(str, srcs), "-lcudart"]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libhier_b200.so")
    if verbose:
        sys.stdout.write(res.stdout + res.stderr)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, force=True)
    print(LIB)

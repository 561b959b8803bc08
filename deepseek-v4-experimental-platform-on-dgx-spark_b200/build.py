"""Compile the CUDA library (csrc/lib.cu) for sm_100a into ``libbsgemm.so``, and the host path of the serving
operators (csrc/bind.cpp, against torch's C++ headers) into ``_native.so``.

    python <package dir>/build.py            # writes both into <package dir>

The library comes first and needs nvcc alone; where torch or a C++ compiler is missing the host path is left out,
with a message.

nvcc cross-compiles without a GPU.  No ``--use_fast_math``: the quantisers
rely on IEEE division and RNE conversions to match the reference bit for bit.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc", "lib.cu")
OUT = os.path.join(HERE, "libbsgemm.so")
BIND_SRC = os.path.join(HERE, "csrc", "bind.cpp")
BIND_OUT = os.path.join(HERE, "_native.so")
DEPS = [os.path.join(HERE, "csrc", f) for f in ("lib.cu", "common.cuh", "quant.cu", "dequant.cu", "hc.cu", "attn.cu", "gemm.cu", "gemm_pair.cu", "capi.cu", "moe.cu", "peer.cu", "moe_fused.cu", "gate.cu", "norm.cu", "rope.cu", "kvcache.cu", "cattn.cu", "noalloc.cu")]
DEPS.append(os.path.join(os.path.dirname(HERE), "include", "bsgemm.h"))


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date(out: str = OUT, deps=None) -> bool:
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(d) <= t for d in (DEPS if deps is None else deps) if os.path.exists(d))


def native_versions() -> str:
    """What the host path's binary interface depends on."""
    import sysconfig

    import torch

    return f"torch {torch.__version__} cxx11_abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} python {sysconfig.get_config_var('SOABI')}"


def native_up_to_date() -> bool:
    """Newer than its sources, and built for the torch and Python at hand (kept beside it, in _native.stamp)."""
    try:
        with open(BIND_OUT[:-3] + ".stamp") as f:
            return f.read() == native_versions() and up_to_date(BIND_OUT, [BIND_SRC, DEPS[-1]])
    except FileNotFoundError:
        return False


def build_native(force: bool = False) -> str:
    """The host path: plain C++ against torch and the C ABI's header, no CUDA code."""
    if not force and native_up_to_date():
        return BIND_OUT
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cuda_include = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", BIND_SRC, "-o", BIND_OUT + ".tmp"]
    for d in [*include_paths(), sysconfig.get_paths()["include"], cuda_include]:
        cmd += ["-isystem", d]
    for d in library_paths():
        cmd += ["-L" + d, "-Wl,-rpath," + d]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    os.replace(BIND_OUT + ".tmp", BIND_OUT)
    with open(BIND_OUT[:-3] + ".stamp", "w") as f:
        f.write(native_versions())
    return BIND_OUT


def build(force: bool = False, verbose: bool = False) -> str:
    build_library(force, verbose)
    try:
        build_native(force)
    except (ImportError, FileNotFoundError) as e:       # no torch, no compiler: callers of the C ABI need neither
        print(f"{BIND_OUT} not built, the serving operators of the Python package need it: {e}", file=sys.stderr)
    return OUT


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    cmd = [nvcc(), "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
           "-Xcompiler", "-fPIC", "-shared", "-o", OUT + ".tmp", SRC]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(r.stderr)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

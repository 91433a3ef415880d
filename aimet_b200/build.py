"""Builds the CUDA library in-tree, aimet_b200/lib/libaimet_b200.so (sm_100a only), and beside it the torch side of the
layers, aimet_b200/lib/_torch_layers.so (host code, g++).

Usage: ``python -m aimet_b200.build [--force] [--verbose]``.  nvcc cross-compiles without a GPU.
Flags that matter for parity with the CPU reference: ``-fmad=false`` (no FMA contraction) and no fast-math.
"""
from __future__ import annotations

import os
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
LIB_DIR = os.path.join(_HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libaimet_b200.so")
SOURCES = ["capi.cu", "qdq_kernels.cu", "stats_kernels.cu", "tfe_search.cu", "v2_hist.cu", "linear.cu", "tensor_gemm.cu", "layer_norm.cu"]
HEADERS = ["common.cuh", "activation.cuh", "tensor_core.cuh", "encoding_math.cuh", "kernels.h", os.path.join("..", "..", "include", "aimet_b200.h")]

TORCH_PATH = os.path.join(LIB_DIR, "_torch_layers.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_layers.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-fmad=false",
    "-Xcompiler", "-fPIC,-O2,-ffp-contract=off",
    "-shared",
    "--threads", "0",   # the sources side by side
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def needs_build(target: str = LIB_PATH, deps=None) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = deps or [os.path.join(CSRC, s) for s in SOURCES + HEADERS]
    return any(os.path.getmtime(d) > t for d in deps + [os.path.abspath(__file__)])


def _torch_tag() -> str:
    """What the torch side's binary depends on beside its source."""
    import torch
    return f"torch {torch.__version__}, {sys.implementation.cache_tag}, cxx11 abi {int(torch.compiled_with_cxx11_abi())}"


def _torch_tag_path() -> str:
    return os.path.splitext(TORCH_PATH)[0] + ".built_for"


def torch_side_is_foreign(unknown: bool = True) -> bool:
    """Whether the torch side was built for another torch or Python than this one (its class layouts may differ);
    ``unknown`` if nothing beside it says what it was built for."""
    try:
        with open(_torch_tag_path(), encoding="utf-8") as f:
            return f.read() != _torch_tag()
    except FileNotFoundError:
        return unknown


def build_torch(force: bool = False, verbose: bool = False) -> str:
    """The autograd functions of :mod:`aimet_b200.v2.nn`; against the torch that is installed."""
    if not force and not needs_build(TORCH_PATH, [TORCH_SOURCE, os.path.join(CSRC, HEADERS[-1])]) and not torch_side_is_foreign():
        return TORCH_PATH
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    os.makedirs(LIB_DIR, exist_ok=True)
    cuda = os.path.dirname(os.path.dirname(_nvcc())) if os.path.isabs(_nvcc()) else "/usr/local/cuda"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_torch_layers",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    for d in cpp_extension.include_paths() + [sysconfig.get_paths()["include"], os.path.join(cuda, "include")]:
        cmd += ["-isystem", d]
    cmd += [TORCH_SOURCE, "-o", TORCH_PATH]
    for d in cpp_extension.library_paths():
        cmd += ["-L" + d]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("g++ failed building _torch_layers.so")
    with open(_torch_tag_path(), "w", encoding="utf-8") as f:
        f.write(_torch_tag())
    return TORCH_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    build_torch(force, verbose)
    if not force and not needs_build():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    cmd = [_nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + \
          [os.path.join(CSRC, s) for s in SOURCES] + ["-o", LIB_PATH]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed building libaimet_b200.so")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))

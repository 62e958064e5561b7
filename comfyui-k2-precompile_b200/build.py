"""Builds libk2b (all CUDA kernels + the C ABI) for sm_100a, and the torch
binding of the conditioning operators on top of it, in-tree.

    python comfyui-k2-precompile_b200/build.py [--force]

Output: comfyui-k2-precompile_b200/k2b/_lib/libk2b.so and _bind.so (git-ignored;
they travel with the working tree).  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "k2b", "_lib", "libk2b.so")
BIND = os.path.join(HERE, "k2b", "_lib", "_bind.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-shared",
]


BIND_SRC = os.path.join(CSRC, "torch_bind.cpp")
HEADER = os.path.join(INCLUDE, "k2b.h")


def sources():
    return sorted(s for s in glob.glob(os.path.join(CSRC, "*")) if s != BIND_SRC) + [HEADER]


def _newer(out: str, srcs) -> bool:
    return os.path.exists(out) and all(os.path.getmtime(s) <= os.path.getmtime(out) for s in srcs)


def up_to_date() -> bool:
    return _newer(OUT, sources())


def bind_up_to_date() -> bool:
    return _newer(BIND, [BIND_SRC, HEADER])


def build_bind() -> None:
    """Host code only: g++ against this interpreter's torch."""
    import torch

    root = os.path.dirname(torch.__file__)
    libdir = os.path.dirname(OUT)
    tmp = BIND + ".tmp"
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
         f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         "-I" + os.path.join(root, "include"), "-I" + sysconfig.get_paths()["include"],
         "-I" + os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), BIND_SRC, "-o", tmp,
         "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
         "-L" + libdir, "-l:libk2b.so", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(tmp, BIND)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        os.makedirs(os.path.dirname(OUT), exist_ok=True)
        tmp = OUT + ".tmp"
        cmd = [NVCC, *FLAGS, "-o", tmp, os.path.join(CSRC, "k2b_lib.cu")]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        subprocess.run(cmd, check=True)
        os.replace(tmp, OUT)
    if force or not bind_up_to_date():
        build_bind()
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

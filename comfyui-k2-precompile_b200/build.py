"""Builds libk2b (all CUDA kernels + the C ABI) for sm_100a, and the torch
binding of the conditioning operators on top of it, in-tree.

    python comfyui-k2-precompile_b200/build.py [--force]

Output: comfyui-k2-precompile_b200/k2b/_lib/libk2b.so and, for each Python and
torch that builds it, a _bind.<ABI>.so (git-ignored; they travel with the working
tree).  libk2b needs nvcc alone, which cross-compiles without a GPU; the binding
needs g++, torch and Python's headers, and is left out where those are missing
(a host of the C entries does not need it).
"""
from __future__ import annotations

import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "k2b", "_lib", "libk2b.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
NVCC = os.path.abspath(shutil.which(NVCC) or NVCC)
CUDA_INCLUDE = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")

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


def bind_path() -> str:
    """Where the binding for this Python and torch goes (k2b/_native.py names it)."""
    spec = importlib.util.spec_from_file_location("_k2b_native", os.path.join(HERE, "k2b", "_native.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod.bind_path()


def bind_up_to_date() -> bool:
    return _newer(bind_path(), [BIND_SRC, HEADER])


def bind_missing() -> str:
    """What this host lacks to build the binding, or nothing."""
    if importlib.util.find_spec("torch") is None:
        return "torch"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers"
    return "" if shutil.which("g++") else "g++"


def build_lib(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        os.makedirs(os.path.dirname(OUT), exist_ok=True)
        tmp = OUT + ".tmp"
        cmd = [NVCC, *FLAGS, "-o", tmp, os.path.join(CSRC, "k2b_lib.cu")]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        subprocess.run(cmd, check=True)
        os.replace(tmp, OUT)
    return OUT


def build_bind(force: bool = False) -> str:
    """Host code only: g++ against this interpreter's torch, on a built libk2b."""
    out = bind_path()
    if not force and bind_up_to_date():
        return out
    import torch

    root = os.path.dirname(torch.__file__)
    tmp = out + ".tmp"
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
         f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         "-I" + os.path.join(root, "include"), "-I" + sysconfig.get_paths()["include"], "-I" + CUDA_INCLUDE,
         BIND_SRC, "-o", tmp,
         "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
         "-L" + os.path.dirname(OUT), "-l:libk2b.so", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(tmp, out)
    return out


def build(force: bool = False, verbose: bool = False) -> str:
    build_lib(force, verbose)
    missing = bind_missing()
    if missing:
        print(f"torch binding not built: {missing} not found", file=sys.stderr)
    else:
        build_bind(force)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

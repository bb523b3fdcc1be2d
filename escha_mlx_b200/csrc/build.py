"""Builds libescha_b200.so (sm_100a) in-tree with nvcc, and the binding of the decode step's
operators with the host compiler.

    python -m escha_mlx_b200.csrc.build [--force] [--verbose]

The library is a plain C-ABI shared object (see include/escha_b200.h); it links
the CUDA runtime statically and has no Python or torch dependency.  The binding
(csrc/bind.cpp) is a Python extension over torch's C++ headers that calls the
library through the addresses it is given.
"""
from __future__ import annotations

import concurrent.futures
import glob
import os
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
LIB = os.path.join(PKG, "libescha_b200.so")
BINDING = os.path.join(PKG, "_decode.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    # no --use_fast_math: fp16 adds and the transform multiplies are rounding points
]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "*.cu")))


def stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(HERE, "*.cuh")) + glob.glob(os.path.join(HERE, "*.h"))
    deps.append(os.path.join(os.path.dirname(PKG), "include", "escha_b200.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed building {cmd[-1]}")
    if verbose:
        print(res.stdout + res.stderr)


def build_binding(force: bool = False, verbose: bool = False) -> str:
    source = os.path.join(HERE, "bind.cpp")
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) >= os.path.getmtime(source):
        return BINDING
    import torch
    from torch.utils import cpp_extension
    include = [f"-I{d}" for d in [*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
                                  os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")]]
    lib_dir = os.path.join(os.path.dirname(torch.__file__), "lib")
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *include, source,
          f"-L{lib_dir}", f"-Wl,-rpath,{lib_dir}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda",
          "-ltorch", "-ltorch_python", "-o", BINDING], verbose)
    return BINDING


def build(force: bool = False, verbose: bool = False) -> str:
    build_binding(force, verbose)
    if not force and not stale():
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    ptxas = ["-Xptxas", "-v"] if verbose else []
    with tempfile.TemporaryDirectory() as tmp:
        # one compiler per source, as many at a time as there are cores
        objects = {src: os.path.join(tmp, os.path.basename(src) + ".o") for src in sources()}
        with concurrent.futures.ThreadPoolExecutor(os.cpu_count() or 1) as pool:
            jobs = [pool.submit(_run, [nvcc, *ptxas, *[f for f in NVCC_FLAGS if f != "-shared"], "-c", src,
                                       "-o", obj], verbose) for src, obj in objects.items()]
            for job in jobs:
                job.result()
        _run([nvcc, *NVCC_FLAGS, *objects.values(), "-o", LIB], verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(LIB)

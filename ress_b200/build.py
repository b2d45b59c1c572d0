"""Builds libress_sm100.so in-tree with nvcc for sm_100a, and _host.so, the
Python module that checks and launches the streaming calls, with g++ against
torch's headers.

Run as ``python -m ress_b200.build`` (or through ``__graft_entry__.build()``).
The library is the product's only compute path; nothing else is compiled
at import time."""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = [os.path.join(HERE, "csrc", f) for f in ("capi.cu", "score.cu", "select.cu", "attn.cu", "noalloc.cu",
                                                "prologue.cu", "cache.cu", "cache_attn.cu", "cache_attn_tc.cu", "int8.cu")]
OUT = os.path.join(HERE, "libress_sm100.so")
HOST_SRC = os.path.join(HERE, "csrc", "host.cpp")
HOST_OUT = os.path.join(HERE, "_host.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "--threads", "0", "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-shared",
    "-I", os.path.join(ROOT, "include"),
]


def needs_build() -> bool:
    if not os.path.exists(OUT) or not os.path.exists(HOST_OUT):
        return True
    t = min(os.path.getmtime(OUT), os.path.getmtime(HOST_OUT))
    deps = SRC + [HOST_SRC] + [os.path.join(HERE, "csrc", h) for h in ("common.cuh", "prologue.cuh", "tcgen05.cuh", "cache.cuh",
                                                       "cache_attn.cuh")]
    deps.append(os.path.join(ROOT, "include", "ress_sm100.h"))
    return any(os.path.getmtime(p) > t for p in deps)


def build_host(verbose: bool = False) -> str:
    import torch
    from torch.utils import cpp_extension as ext

    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++20", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{d}" for d in [*ext.include_paths(), sysconfig.get_paths()["include"],
                                      os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]),
           HOST_SRC, f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-o", HOST_OUT]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return HOST_OUT


def build(verbose: bool = False, ptxas_info: bool = False) -> str:
    cmd = [NVCC, *FLAGS, *SRC, "-o", OUT]
    if ptxas_info:
        cmd.insert(1, "-Xptxas=-v")
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    build_host(verbose)
    return OUT


if __name__ == "__main__":
    build(verbose=True, ptxas_info="-v" in sys.argv)

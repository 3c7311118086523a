"""Builds libbasedxl_b200.so in-tree with nvcc for sm_100a, and _native.so beside it.

    python -m basedxl_b200.build [--force] [--verbose]

The library is plain CUDA C++ behind a C ABI (include/basedxl_b200.h); it links
only against the CUDA runtime.  The driver API entry point it needs for TMA
descriptors is resolved at run time.  _native.so holds the native wrappers of the
training operators: host code against PyTorch's headers, linked to the library.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libbasedxl_b200.so")
NATIVE = os.path.join(PKG, "_native.so")
NATIVE_SOURCE = os.path.join(CSRC, "bindings.cpp")
SOURCES = ["bxl_host.cu", "gemm_conv.cu", "groupnorm.cu", "attention.cu", "elementwise.cu", "layernorm.cu", "linear.cu", "comm.cu"]
HEADERS = ["bxl_common.cuh", "bxl_host.h", "bxl_types.cuh", "bxl_act.cuh", os.path.join("..", "..", "include", "basedxl_b200.h")]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: the CUDA extension cannot be built")
    return nvcc


def _older(target: str, deps) -> bool:
    return not os.path.exists(target) or any(os.path.getmtime(d) > os.path.getmtime(target) for d in deps)


def needs_build() -> bool:
    return _older(LIB, [os.path.join(CSRC, s) for s in SOURCES + HEADERS])


def build_native() -> str:
    import torch

    root = os.path.dirname(os.path.abspath(torch.__file__))
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
                os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in includes), NATIVE_SOURCE, "-o", NATIVE, f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch",
           "-lc10_cuda", "-lc10", f"-L{PKG}", "-lbasedxl_b200", "-Wl,-rpath,$ORIGIN"]
    subprocess.check_call(cmd)
    return NATIVE


def build(force: bool = False, verbose: bool = False) -> str:
    if force or needs_build():
        _build_library(verbose)
    if force or _older(NATIVE, [NATIVE_SOURCE, os.path.join(CSRC, HEADERS[-1]), LIB]):
        build_native()
    return LIB


def _build_library(verbose: bool) -> None:
    nvcc = _nvcc()
    objs = []
    obj_dir = os.path.join(PKG, "build")
    os.makedirs(obj_dir, exist_ok=True)
    procs = []
    for s in SOURCES:
        obj = os.path.join(obj_dir, s.replace(".cu", ".o"))
        cmd = [nvcc, *NVCC_FLAGS, "-c", os.path.join(CSRC, s), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        procs.append((s, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = False
    for s, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode != 0:
            sys.stderr.write(f"--- {s} ---\n{out}\n")
        failed |= p.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    subprocess.check_call([nvcc, "-shared", "-o", LIB, *objs, "-lcudart"])


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))

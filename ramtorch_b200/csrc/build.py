"""Build ``ramtorch_b200/librt_b200.so`` in-tree with nvcc for sm_100a.

    python -m ramtorch_b200.csrc.build [--force] [--verbose]

The library is plain CUDA C++ behind a C ABI (include/rt_b200.h): no torch headers, no pybind.
It links the shared CUDA runtime so that, inside a PyTorch process, it uses the runtime
instance torch already loaded (same primary contexts, streams and current device).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
OUT = os.path.join(PKG, "librt_b200.so")
OBJ = os.path.join(HERE, "_obj")
SOURCES = ["adamw_sr.cu", "offload.cu", "microscale.cu", "mx_gemm.cu"]
DEPS = SOURCES + ["philox.cuh", "mx_common.cuh", "tc05.cuh", "rt_internal.h", os.path.join(ROOT, "include", "rt_b200.h")]


def nvcc_path() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    if os.path.exists(cand):
        return cand
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found: librt_b200.so cannot be built")
    return found


def stale() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    return any(os.path.getmtime(os.path.join(HERE, d)) > t for d in DEPS)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not stale():
        return OUT
    nvcc = nvcc_path()
    cuda_lib = os.path.join(os.path.dirname(os.path.dirname(nvcc)), "lib64")
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    flags = arch + ["-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-O2,-Wall"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    os.makedirs(OBJ, exist_ok=True)

    def run(cmd):
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
        return res.returncode

    def compile_one(name):      # one translation unit at a time per thread; unchanged ones keep their object
        src, obj = os.path.join(HERE, name), os.path.join(OBJ, name[:-3] + ".o")
        newest = max(os.path.getmtime(os.path.join(HERE, d)) for d in [name] + [d for d in DEPS if not d.endswith(".cu")])
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > newest:
            return 0, obj
        return run([nvcc, *flags, "-c", src, "-o", obj]), obj

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        done = list(pool.map(compile_one, SOURCES))
    link = [nvcc, *arch, "-shared", "-cudart", "shared", "-Xlinker", f"-rpath={cuda_lib}", "-o", OUT + ".tmp"]
    if any(rc for rc, _ in done) or run(link + [obj for _, obj in done]):
        raise RuntimeError("nvcc failed building librt_b200.so")
    os.replace(OUT + ".tmp", OUT)
    return OUT


def _build_module(name: str, src: str, out: str, force: bool, deps=(), cuda: bool = False) -> str:
    """Build an optional host-side helper with g++ against the torch headers of the running interpreter."""
    if not force and os.path.exists(out) and all(os.path.getmtime(out) >= os.path.getmtime(d) for d in (src, *deps)):
        return out
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ce
    gxx = shutil.which("g++")
    if not gxx:
        raise RuntimeError(f"g++ not found: {name}.so cannot be built")
    inc = ce.include_paths() + [sysconfig.get_paths()["include"]]
    libs = ce.library_paths()
    cmd = [gxx, "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-DTORCH_EXTENSION_NAME={name}", "-DTORCH_API_INCLUDE_EXTENSION_H"]
    link = ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10"]
    if cuda:
        inc.append(os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include"))
        link += ["-ltorch_cuda", "-lc10_cuda"]
    cmd += [f"-I{i}" for i in inc] + [src, "-o", out + ".tmp"]
    cmd += [f"-L{d}" for d in libs] + [f"-Wl,-rpath,{d}" for d in libs] + link
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"g++ failed building {name}.so")
    os.replace(out + ".tmp", out)
    return out


FASTSCAN_SRC = os.path.join(HERE, "fastscan.cpp")
FASTSCAN_OUT = os.path.join(PKG, "_fastscan.so")
MXCALL_SRC = os.path.join(HERE, "mxcall.cpp")
MXCALL_OUT = os.path.join(PKG, "_mxcall.so")


def build_fastscan(force: bool = False) -> str:
    """Build ``ramtorch_b200/_fastscan.so``, the host-side helper that walks long parameter lists in
    C++.  It only reads tensor pointers and properties; the optimizer works without it, with
    per-tensor Python passes instead."""
    return _build_module("_fastscan", FASTSCAN_SRC, FASTSCAN_OUT, force)


def build_mxcall(force: bool = False) -> str:
    """Build ``ramtorch_b200/_mxcall.so``, the host side of the microscaled calls in C++ (allocation, current device
    and stream, the call of the C ABI).  ``microscaling`` works without it, through ctypes."""
    return _build_module("_mxcall", MXCALL_SRC, MXCALL_OUT, force, deps=(os.path.join(ROOT, "include", "rt_b200.h"),), cuda=True)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
    print(build_fastscan(force="--force" in sys.argv))
    print(build_mxcall(force="--force" in sys.argv))

"""Builds the CUDA extension in-tree: rapidocrvl_b200/libocrvl_cuda.so.

sm_100a only.  engine.cu is compiled with -fmad=false, which keeps
multiply/add pairs unfused so that the explicit __fmaf_rn calls are the only
fused operations (its kernels restate the reference's CPU rounding step by
step); kvops.cu's operators have no such order to keep.

The torch side of those operators is a second library, _kvops, which links the
first: the C ABI itself needs nothing from torch.
"""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libocrvl_cuda.so")
TORCH_SOURCE = os.path.join(CSRC, "kvops_torch.cpp")
TORCH_LIB = os.path.join(HERE, "_kvops.so")
HEADER = os.path.join(ROOT, "include", "ocrvl_cuda.h")
SOURCES = {"engine.cu": ["-fmad=false"], "kvops.cu": []}  # and the flags of their own

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [*ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-Xptxas", "-v"]


def nvcc() -> str:
    for p in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if p and (os.path.isabs(p) and os.path.exists(p) or not os.path.isabs(p)):
            return p
    return "nvcc"


def older(out: str, files) -> bool:
    return not os.path.exists(out) or any(os.path.getmtime(f) > os.path.getmtime(out) for f in files)


def needs_build() -> bool:
    return older(LIB, [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))] + [HEADER])


def run(cmd, what: str) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"{cmd[0]} failed building {what}")
    return r.stderr


def build_torch(force: bool = False) -> str:
    """The torch side of the paged-cache operators; imports torch."""
    build(force=False)
    if not force and not older(TORCH_LIB, [TORCH_SOURCE, HEADER]):
        return TORCH_LIB
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    dirs = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         *(x for d in dirs for x in ("-isystem", d)), TORCH_SOURCE, "-o", TORCH_LIB + ".tmp", "-L", HERE, "-l:libocrvl_cuda.so",
         "-Wl,-rpath,$ORIGIN", "-L", libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"], "_kvops.so")
    os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    with tempfile.TemporaryDirectory() as tmp:
        objects = {src: os.path.join(tmp, src + ".o") for src in SOURCES}
        with ThreadPoolExecutor() as pool:
            said = pool.map(lambda src: run([nvcc(), *NVCC_FLAGS, *SOURCES[src], "-I", os.path.join(ROOT, "include"), "-c",
                                             os.path.join(CSRC, src), "-o", objects[src]], src), SOURCES)
            for text in said:
                if verbose:
                    sys.stderr.write(text)
        run([nvcc(), *ARCH, "-shared", "-o", LIB + ".tmp", *objects.values()], "libocrvl_cuda.so")
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
    if importlib.util.find_spec("torch"):
        print(build_torch(force="--force" in sys.argv))
    else:  # a host of the C ABI needs nothing else
        print("no torch: _kvops.so not built")

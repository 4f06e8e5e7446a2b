"""Builds the CUDA extension in-tree: rapidocrvl_b200/libocrvl_cuda.so.

sm_100a only.  engine.cu is compiled with -fmad=false, which keeps
multiply/add pairs unfused so that the explicit __fmaf_rn calls are the only
fused operations (its kernels restate the reference's CPU rounding step by
step); kvops.cu's operators have no such order to keep.
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libocrvl_cuda.so")
SOURCES = {"engine.cu": ["-fmad=false"], "kvops.cu": []}  # and the flags of their own

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [*ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-Xptxas", "-v"]


def nvcc() -> str:
    for p in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if p and (os.path.isabs(p) and os.path.exists(p) or not os.path.isabs(p)):
            return p
    return "nvcc"


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))]
    files.append(os.path.join(ROOT, "include", "ocrvl_cuda.h"))
    return any(os.path.getmtime(f) > t for f in files)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    def run(cmd) -> str:
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("nvcc failed building libocrvl_cuda.so")
        return r.stderr

    with tempfile.TemporaryDirectory() as tmp:
        objects = {src: os.path.join(tmp, src + ".o") for src in SOURCES}
        with ThreadPoolExecutor() as pool:
            said = pool.map(lambda src: run([nvcc(), *NVCC_FLAGS, *SOURCES[src], "-I", os.path.join(ROOT, "include"), "-c",
                                             os.path.join(CSRC, src), "-o", objects[src]]), SOURCES)
            for text in said:
                if verbose:
                    sys.stderr.write(text)
        run([nvcc(), *ARCH, "-shared", "-o", LIB + ".tmp", *objects.values()])
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)

"""In-tree build of librzlinear_b200.so (nvcc, sm_100a only).

    python -m rzlinear_b200.build [--force] [--verbose]

The library is plain CUDA C++ behind a C ABI (include/rzlinear_b200.h); it does not link
against PyTorch.  nvcc cross-compiles it on a machine without a GPU.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_PATH = os.path.join(HERE, "librzlinear_b200.so")
SOURCES = ["rz_abi.cu", "rz_simt.cu", "rz_tc.cu", "rz_noalloc.cu", "rz_elementwise.cu", "rz_rows.cu",
           "rz_grouped.cu", "rz_tc_grouped.cu"]
HEADERS = ["rz_common.h", "rz_hash.h", "rz_ptx.cuh", "rz_tc_kernel.cuh", "rz_tc_rows.cuh", "rz_tc_host.h", os.path.join("..", "..", "include", "rzlinear_b200.h")]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, s) for s in SOURCES + HEADERS]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB_PATH
    flags = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]
    if verbose:
        flags += ["-Xptxas", "-v"]

    def run(args):
        return subprocess.run([_nvcc()] + args, capture_output=True, text=True)

    with tempfile.TemporaryDirectory() as tmp:   # one object per source, compiled side by side
        objects = [os.path.join(tmp, s + ".o") for s in SOURCES]
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            done = list(pool.map(run, [flags + ["-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(SOURCES, objects)]))
        if not any(p.returncode for p in done):
            done.append(run(["-shared", "-cudart", "shared", "-Xlinker", "-rpath=/usr/local/cuda/lib64", "-o", LIB_PATH] + objects))
    for proc in done:
        if verbose or proc.returncode:
            sys.stderr.write(proc.stdout + proc.stderr)
    if any(p.returncode for p in done):
        raise RuntimeError("nvcc failed building librzlinear_b200.so")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))

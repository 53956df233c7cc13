"""Builds libw4b200.so (the CUDA kernels + the C ABI) for sm_100a, in-tree.

    python w4a16-dequant-gemm_b200/build.py [--force]

nvcc cross-compiles without a GPU. The library lands in
w4a16-dequant-gemm_b200/lib/ (git-ignored; it travels with the source tree).
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libw4b200.so")
FASTCALL = os.path.join(LIB_DIR, "_w4b_fastcall.so")  # CPython binding of the per-step entries (csrc/fastcall.cpp)
SOURCES = ["abi.cu", "dequant.cu", "gemm_generic.cu", "gemm_stream.cu", "gemm_noalloc.cu", "gemm_tensor.cu", "attn_flash.cu", "attn_mma.cu", "peer_gather.cu", "quantize.cu", "relayout.cu",
           "page_tables.cu", "kv_write_b8.cu", "attn_b8.cu", "attn_b8_chunk.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-shared"]


def _stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(FASTCALL):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(FASTCALL))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(os.path.dirname(HERE), "include", "w4b_abi.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    os.makedirs(LIB_DIR, exist_ok=True)
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-o", LIB] + \
        [os.path.join(CSRC, s) for s in SOURCES]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    if verbose:
        print(r.stderr)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-I" + sysconfig.get_paths()["include"],
           os.path.join(CSRC, "fastcall.cpp"), "-o", FASTCALL, "-L" + LIB_DIR, "-l:libw4b200.so", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed:\n" + r.stdout + r.stderr)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

"""Builds the two sm_100a attention-backward libraries in-tree:

    build/libfmha_bwd_bf16.so   (fmha_bwd_full_py, fmha_bwd_full_stream, ...)
    build/libfmha_bwd_fp16.so   (fmha_bwd_full_fp16, fmha_bwd_full_fp16_stream, ...)

at the repository root, the paths the reference's ctypes host loads
(benchmark_pytorch_final.py:30 loads ./build/libfmha_bwd_bf16.so). nvcc
cross-compiles for sm_100a without a GPU. Run: python build_libs.py [--force]
"""
from __future__ import annotations

import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT = os.path.join(ROOT, "build")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
]

LIBS = {
    "libfmha_bwd_bf16.so": ("fmha_bwd_bf16.cu", "fmha_attn_bf16.cu"),
    "libfmha_bwd_fp16.so": ("fmha_bwd_fp16.cu", "fmha_attn_fp16.cu"),
}


def _sources_mtime() -> float:
    sources = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    return max(os.path.getmtime(f) for f in sources + [os.path.join(ROOT, "include", "fmha_bwd.h")])


def build(force: bool = False, verbose: bool = False) -> list[str]:
    os.makedirs(OUT, exist_ok=True)
    newest = _sources_mtime()
    stale = [lib for lib in LIBS if force or not os.path.exists(os.path.join(OUT, lib))
             or os.path.getmtime(os.path.join(OUT, lib)) < newest]
    extra = ["-Xptxas=-v"] if verbose else []
    # one object per source, all of them at once, then one link per library
    jobs = [(src, os.path.join(OUT, src[:-3] + ".o")) for lib in stale for src in LIBS[lib]]
    running = [(src, subprocess.Popen([NVCC, *FLAGS, *extra, "-c", "-o", obj, os.path.join(CSRC, src)], cwd=CSRC))
               for src, obj in jobs]
    failed = [src for src, proc in running if proc.wait() != 0]
    if failed:
        raise RuntimeError(f"nvcc failed on {', '.join(failed)}")
    for lib in stale:
        objs = [os.path.join(OUT, src[:-3] + ".o") for src in LIBS[lib]]
        subprocess.run([NVCC, *FLAGS, "-shared", "-o", os.path.join(OUT, lib), *objs], check=True, cwd=CSRC)
    return [os.path.join(OUT, lib) for lib in LIBS]


if __name__ == "__main__":
    for p in build(force="--force" in sys.argv, verbose="-v" in sys.argv):
        print(p)

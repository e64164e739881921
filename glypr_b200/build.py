"""Build libglypr_cuda.so in-tree with nvcc for sm_100a (no GPU needed to compile)."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libglypr_cuda.so")
SOURCES = ["glypr_cuda.cu", "op_rows_f32.cu", "op_rows_f16.cu", "op_rows_bf16.cu", "op_rows.cu", "op_linear.cu",
           "gguf.cpp", "engine.cpp", "tokenizer.cpp"]
HEADERS = ["common.cuh", "gemm.cuh", "q8gemm.cuh", "attention_tc.cuh", "attention_d512.cuh", "attention_pair.cuh", "rowops.cuh", "gguf.h", "ple.cuh",
           "rowquant.cuh", "op_rows.cuh", "linear.cuh", "linear_any.cuh",
           "linear_rows.cuh", "linear_tc.cuh", "linear_splitk.cuh", "operators.h", "unicode_case.inc"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC,-O3", "-I", os.path.join(ROOT, "include"), "-I", CSRC]


def commands(obj_dir, extra=()) -> tuple:
    """One compile command per source, and the link command."""
    objs = [os.path.join(obj_dir, s + ".o") for s in SOURCES]
    compiles = [[nvcc(), *FLAGS, "-c", os.path.join(CSRC, s), "-o", o, *extra] for s, o in zip(SOURCES, objs)]
    return compiles, [nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *objs, "-o", LIB,
                      "-cudart", "static", "-lpthread", "-ldl", "-lrt"]


def stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS] + [os.path.join(ROOT, "include", "glypr_cuda.h")]
    return any(os.path.getmtime(p) > t for p in deps if os.path.exists(p))


def build(force: bool = False, verbose: bool = False, extra=()) -> str:
    if force or stale():
        with tempfile.TemporaryDirectory() as obj_dir:
            compiles, link = commands(obj_dir, extra)

            def run(cmd):
                if verbose:
                    print(" ".join(cmd), flush=True)
                subprocess.run(cmd, check=True)
            with ThreadPoolExecutor(max_workers=min(len(compiles), os.cpu_count() or 1)) as pool:
                list(pool.map(run, compiles))
            run(link)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True,
          extra=["-Xptxas", "-v"] if "--ptxas" in sys.argv else [])

"""Build the perseus-b200 CUDA library in-tree: perseus_b200/libpcb200.so (sm_100a).

One nvcc invocation per translation unit (objects under perseus_b200/_build/), then one shared link. Rebuilds only
what changed. Cross-compiles without a GPU.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libpcb200.so")
SOURCES = ["ntt.cu", "elem.cu", "pt.cu", "ks.cu", "regen.cu", "keys.cu", "table.cu", "evaluator.cu", "probe.cu", "wire.cu", "elem_multi.cu", "cts.cu", "clear.cu", "clear_gemm.cu", "clear_attn.cu"]
HEADERS = ["arith.cuh", "chacha.cuh", "keyregen.cuh", "kernels.h", "host_math.h", "ntt_pipe.cuh", "clear.h", "clear_gemm.h", "mma.cuh"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2,-ffp-contract=off",
    "-Xptxas", "-warn-spills",
    "-ccbin", "g++",
]


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose=False):
    os.makedirs(BUILD, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(ROOT, "include", "pcb200.h")]
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src.replace(".cu", ".o"))
        objs.append(o)
        if _stale(o, [s] + hdrs):
            cmd = [NVCC] + FLAGS + ["-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd))
            subprocess.run(cmd, check=True)
    if _stale(LIB, objs):
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB] + objs + ["-lcudart"]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))

"""Builds libcoli_cuda_backend.so (sm_100a only) in-tree with nvcc."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libcoli_cuda_backend.so")

_HEADER = os.path.join("..", "..", "include", "peregrine_b200.h")
# translation units with what they include
SOURCES = {
    "backend.cu": ["ptx.cuh", "kernels.cuh", "kernels_mma.cuh", "kernels_tile.cuh", "kernels_tcgen05.cuh", "kernels_fold.cuh",
                   "kernels_decode.cuh", "kernels_block.cuh", "kernels_ep.cuh", "backend_ep.inc", "w4_layout.h",
                   "expert_route.h", "w4_host.h", "backend_layer.inc", "backend_pipe.inc", "backend_noalloc.inc", "ctx.h",
                   _HEADER],
    "attn.cu": ["ptx.cuh", "ctx.h", "kernels_norm_rope.cuh", "kernels_attn.cuh", "kernels_attn_tc.cuh", "kernels_evict.cuh", "kv_overlap.h", _HEADER],
    "w4_host.cpp": ["w4_host.h", "w4_layout.h"],
}

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    # the CPU reference never contracts a*b+c; neither may the device code
    "-fmad=false", "-prec-div=true", "-prec-sqrt=true",
    "-Xcompiler", "-fPIC,-fvisibility=hidden,-O2",
]
LINK_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-cudart", "static"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA backend cannot be built")


def _stale(target: str, inputs) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(p) > t for p in inputs)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the translation units that are out of date, side by side, and links them."""
    files = [os.path.join(CSRC, f) for s, deps in SOURCES.items() for f in [s] + deps]
    if not (force or _stale(LIB, files)):
        return LIB
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    objs, jobs = [], []
    for src, deps in SOURCES.items():
        obj = os.path.join(objdir, src + ".o")
        objs.append(obj)
        if force or _stale(obj, [os.path.join(CSRC, f) for f in [src] + deps]):
            cmd = [_nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", obj, src]
            jobs.append((cmd, obj, subprocess.Popen(cmd, cwd=CSRC)))
    failed = None
    for cmd, obj, job in jobs:
        if job.wait() != 0:
            failed = subprocess.CalledProcessError(job.returncode, cmd)
            if os.path.exists(obj):
                os.remove(obj)
    if failed:
        raise failed
    subprocess.check_call([_nvcc()] + LINK_FLAGS + ["-o", LIB] + objs, cwd=CSRC)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

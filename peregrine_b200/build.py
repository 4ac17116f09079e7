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


def _stamp(target: str) -> str:
    return os.path.join(HERE, "build", os.path.basename(target) + ".cmd")


def _command(target: str):
    """What ``target`` was made by, or None."""
    try:
        with open(_stamp(target)) as f:
            return f.read()
    except FileNotFoundError:
        return None


def _remember(target: str, command: str) -> None:
    with open(_stamp(target), "w") as f:
        f.write(command)


def _forget(target: str) -> None:
    for p in (_stamp(target), target):
        if os.path.exists(p):
            os.remove(p)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the translation units that are out of date, side by side, and links them.  A unit is so when a file of its is newer
    or when it was compiled by another command; ``verbose`` compiles all of them, to print what each kernel takes."""
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    stale = []
    for src, deps in SOURCES.items():
        obj = os.path.join(objdir, src + ".o")
        command = " ".join(NVCC_FLAGS + ["-c", src])
        if force or verbose or _stale(obj, [os.path.join(CSRC, f) for f in [src] + deps]) or _command(obj) != command:
            stale.append((src, obj, command))
    objs = [os.path.join(objdir, src + ".o") for src in SOURCES]
    link = " ".join(LINK_FLAGS)
    if not stale and not _stale(LIB, objs) and _command(LIB) == link:
        return LIB
    nvcc = _nvcc()
    jobs = []
    for src, obj, command in stale:
        _forget(obj)
        cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", obj, src]
        jobs.append((cmd, obj, command, subprocess.Popen(cmd, cwd=CSRC)))
    failed = None
    for cmd, obj, command, job in jobs:
        if job.wait() == 0:
            _remember(obj, command)
        else:
            failed = subprocess.CalledProcessError(job.returncode, cmd)
    if failed:
        raise failed
    subprocess.check_call([nvcc] + LINK_FLAGS + ["-o", LIB + ".new"] + objs, cwd=CSRC)
    os.replace(LIB + ".new", LIB)  # a process that has the old one loaded keeps it
    _remember(LIB, link)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

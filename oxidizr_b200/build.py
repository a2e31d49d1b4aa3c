"""Builds liboxz_dpstep.so in-tree with nvcc for sm_100a (cross-compiles without a GPU)."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liboxz_dpstep.so")
SOURCES = ["oxz_kernels.cu", "oxz_noalloc.cu", "oxz_loader.cu", "oxz_embed.cu", "oxz_head.cu", "oxz_plan.cpp", "oxz_step.cpp", "oxz_comm.cpp", "oxz_host.cpp", "oxz_checkpoint.cpp", "oxz_meta.cpp", "oxz_launch.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA kernels cannot be built")


def _host_compiler() -> list[str]:
    # A wrapper compiler on PATH may lack pieces nvcc needs; the system g++ is the safe choice when present.
    return ["-ccbin", "/usr/bin/g++"] if os.path.exists("/usr/bin/g++") else []


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "oxz_dpstep.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    # one nvcc per source, side by side: the kernels' template instances are most of the time
    flags = [*ARCH, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-Wall,-Wextra", *_host_compiler(), *(["-Xptxas=-v"] if verbose else [])]
    with tempfile.TemporaryDirectory() as out, ThreadPoolExecutor(os.cpu_count() or 1) as pool:
        objects = [os.path.join(out, s + ".o") for s in SOURCES]
        cmds = [[_nvcc(), *flags, "-c", "-o", o, os.path.join(CSRC, s)] for s, o in zip(SOURCES, objects)]
        if verbose:
            print("\n".join(" ".join(c) for c in cmds))
        list(pool.map(lambda c: subprocess.run(c, check=True), cmds))
        subprocess.run([_nvcc(), *ARCH, "-shared", *_host_compiler(), "-cudart", "static", "-o", LIB, *objects, "-ldl"], check=True)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)

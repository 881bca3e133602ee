"""Build step for libaljabr_blackwell.so (nvcc, sm_100a, in-tree).

``python -m aljabr_b200.build`` compiles every ``csrc/*.cu`` translation unit
into ``aljabr_b200/libaljabr_blackwell.so`` with relocatable device code (but
for WHOLE) and the CUDA runtime linked statically, so the library depends on
nothing but the driver.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaljabr_blackwell.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2",
    "--expt-relaxed-constexpr",
    "-I", os.path.join(ROOT, "include"),
]
# Compiled by themselves: ptxas ignores setmaxnreg in relocatable device code, whose registers a caller must be able to
# count on.  What these share with the other files they are given as arguments.
WHOLE = ("kv4_tree.cu",)


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) \
        + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return any(os.path.getmtime(p) > t for p in deps)


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    if not force and not _stale():
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    flags = [*NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose_ptxas else [])]
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(os.cpu_count()) as pool:
        def compile_one(src: str) -> str:
            obj = os.path.join(tmp, os.path.basename(src) + ".o")
            rdc = "false" if os.path.basename(src) in WHOLE else "true"
            subprocess.check_call([nvcc, *flags, f"-rdc={rdc}", "-c", src, "-o", obj])
            return obj
        objects = list(pool.map(compile_one, sources()))
        subprocess.check_call([nvcc, *flags, "-rdc=true", "-shared", *objects, "-o", LIB + ".tmp", "-ldl"])
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose_ptxas="--ptxas-v" in sys.argv))

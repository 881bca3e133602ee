"""Build step for libaljabr_blackwell.so (nvcc, sm_100a, in-tree).

``python -m aljabr_b200.build`` compiles every ``csrc/*.cu`` translation unit
into ``aljabr_b200/libaljabr_blackwell.so`` with relocatable device code (but
for WHOLE) and the CUDA runtime linked statically, so the library depends on
nothing but the driver.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaljabr_blackwell.so")
CALLS = os.path.join(HERE, "tensor_calls.so")     # torch tensors to the C-ABI, for kv4.py

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
    if not os.path.exists(LIB) or not os.path.exists(CALLS):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(CALLS))
    deps = sources() + [os.path.join(CSRC, "tensor_calls.cpp")] + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) \
        + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return any(os.path.getmtime(p) > t for p in deps)


def _build_calls(tmp: str) -> str:
    """tensor_calls.cpp against the installed torch's headers (no CUDA code)."""
    import sysconfig
    import torch
    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(os.environ.get("NVCC", "nvcc")))))
    obj = os.path.join(tmp, "tensor_calls.o")
    subprocess.check_call([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-c", os.path.join(CSRC, "tensor_calls.cpp"),
                           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DALJ_TORCH="{torch.__version__}"', "-I", inc,
                           "-I", os.path.join(inc, "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"],
                           "-I", os.path.join(cuda, "include"), "-o", obj])
    return obj


def _link_calls(obj: str) -> str:
    import torch
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    subprocess.check_call([os.environ.get("CXX", "g++"), "-shared", obj, "-o", CALLS + ".tmp", "-Wl,-rpath,$ORIGIN", "-L", HERE,
                           "-l:" + os.path.basename(LIB), "-L", libs, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10"])
    return CALLS + ".tmp"


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
        calls = pool.submit(_build_calls, tmp)
        objects = list(pool.map(compile_one, sources()))
        subprocess.check_call([nvcc, *flags, "-rdc=true", "-shared", *objects, "-o", LIB + ".tmp", "-ldl"])
        os.replace(LIB + ".tmp", LIB)
        os.replace(_link_calls(calls.result()), CALLS)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose_ptxas="--ptxas-v" in sys.argv))

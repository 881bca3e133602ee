"""Build step for libaljabr_blackwell.so (nvcc, sm_100a, in-tree).

``python -m aljabr_b200.build`` compiles every ``csrc/*.cu`` translation unit
into ``aljabr_b200/libaljabr_blackwell.so`` with relocatable device code (but
for WHOLE) and the CUDA runtime linked statically, so the library depends on
nothing but the driver.  nvcc cross-compiles without a GPU.  Where a torch for
CUDA, its headers, Python's and a C++ compiler are there, it also builds
``aljabr_b200/tensor_calls.so``, which kv4.py can do without.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaljabr_blackwell.so")
CALLS = os.path.join(HERE, "tensor_calls.so")     # torch tensors to the C-ABI, for kv4.py
NVCC, CXX = os.environ.get("NVCC", "nvcc"), os.environ.get("CXX", "g++")

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


def _newer(made: str, deps: list[str]) -> bool:
    return not os.path.exists(made) or any(os.path.getmtime(p) > os.path.getmtime(made) for p in deps)


def _stale() -> bool:
    return _newer(LIB, sources() + [p for e in ("cuh", "h") for p in glob.glob(os.path.join(CSRC, "*." + e))] +
                  glob.glob(os.path.join(ROOT, "include", "*.h")))


def _torch():
    """The installed torch, if it can be built against: None, and why."""
    try:
        import torch
    except ImportError as e:
        return None, str(e)
    inc = os.path.join(os.path.dirname(torch.__file__), "include", "ATen", "ATen.h")
    py = os.path.join(sysconfig.get_paths()["include"], "Python.h")
    for need in (inc, py):
        if not os.path.exists(need):
            return None, f"{need} is missing"
    if torch.version.cuda is None:
        return None, "this torch has no CUDA"
    return (torch, "") if shutil.which(CXX) else (None, f"{CXX} is missing")


def _mark(torch) -> str:      # in the file, so that another torch's is known without loading it
    return f"tensor_calls for torch {torch.__version__}"


def _calls_stale(torch) -> bool:
    if _newer(CALLS, [os.path.join(CSRC, "tensor_calls.cpp"), os.path.join(ROOT, "include", "aljabr_blackwell.h")]):
        return True
    with open(CALLS, "rb") as f:
        return _mark(torch).encode() + b"\0" not in f.read()


def _build_calls(torch) -> None:
    """tensor_calls.cpp against the installed torch (no CUDA code)."""
    base = os.path.dirname(torch.__file__)
    inc, libs = os.path.join(base, "include"), os.path.join(base, "lib")
    nvcc = shutil.which(NVCC)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc))) if nvcc else "/usr/local/cuda"
    with tempfile.TemporaryDirectory() as tmp:
        obj = os.path.join(tmp, "tensor_calls.o")
        subprocess.check_call([CXX, "-O2", "-std=c++17", "-fPIC", "-c", os.path.join(CSRC, "tensor_calls.cpp"),
                               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                               f'-DALJ_TORCH="{torch.__version__}"', f'-DALJ_MARK="{_mark(torch)}"', "-I", inc,
                               "-I", os.path.join(inc, "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"],
                               "-I", os.path.join(cuda, "include"), "-o", obj])
        subprocess.check_call([CXX, "-shared", obj, "-o", CALLS + ".tmp", "-Wl,-rpath,$ORIGIN", "-L", HERE,
                               "-l:" + os.path.basename(LIB), "-L", libs, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10"])
    os.replace(CALLS + ".tmp", CALLS)


def _build_lib(verbose_ptxas: bool) -> None:
    flags = [*NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose_ptxas else [])]
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(os.cpu_count()) as pool:
        def compile_one(src: str) -> str:
            obj = os.path.join(tmp, os.path.basename(src) + ".o")
            rdc = "false" if os.path.basename(src) in WHOLE else "true"
            subprocess.check_call([NVCC, *flags, f"-rdc={rdc}", "-c", src, "-o", obj])
            return obj
        objects = list(pool.map(compile_one, sources()))
        subprocess.check_call([NVCC, *flags, "-rdc=true", "-shared", *objects, "-o", LIB + ".tmp", "-ldl"])
    os.replace(LIB + ".tmp", LIB)


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    """The library, and where torch can be built against tensor_calls.so, which only saves its callers host time."""
    if force or _stale():
        _build_lib(verbose_ptxas)
    torch, why = _torch()
    if torch is None:
        print(f"tensor_calls.so is not built ({why}): calls of kv4.py go through ctypes", file=sys.stderr)
    elif force or _calls_stale(torch):
        try:
            _build_calls(torch)
        except subprocess.CalledProcessError as e:
            warnings.warn(f"tensor_calls.so could not be built (status {e.returncode}): calls of kv4.py go through ctypes", RuntimeWarning,
                          stacklevel=2)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose_ptxas="--ptxas-v" in sys.argv))

"""Builds ``libconvrot.so`` (the sm_100a kernels and their C ABI) in-tree with nvcc, and ``_fast-*.so`` (the attention
operators' common calls in compiled form, for this Python and torch) with the host compiler.

``python -m hyperflow_h3_flash_b200.build`` or ``build()`` from Python. Both are written next to this file so
that they travel with a copy of the repository; nothing is installed elsewhere.
"""

from __future__ import annotations

import os
import platform
import shutil
import subprocess
import sys
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libconvrot.so")
SOURCES = sorted(os.path.join(HERE, "csrc", name) for name in os.listdir(os.path.join(HERE, "csrc"))
                 if name.endswith((".cu", ".cuh", ".h")))
FAST_SOURCE = os.path.join(HERE, "csrc", "fast_call.cpp")
HEADER = os.path.join(os.path.dirname(HERE), "include", "convrot.h")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def stale(built: str = LIB, sources: list[str] | None = None) -> bool:
    if not os.path.exists(built):
        return True
    when = os.path.getmtime(built)
    return any(os.path.getmtime(src) > when for src in (SOURCES if sources is None else sources) + [HEADER])


def fast_path() -> str:
    """The module of the common calls.  It depends on the binary interfaces of Python and of torch: their versions are
    part of its name, so that a module of other ones is neither taken nor thought up to date."""
    import torch

    return os.path.join(HERE, f"_fast-{sys.implementation.cache_tag}-{platform.machine()}-torch{torch.__version__}.so")


def build_fast(force: bool = False, verbose: bool = False) -> str:
    """Compiles the Python module of the common calls (it links against torch and takes the library's entries at run
    time); returns its path."""
    built = fast_path()
    if not force and not stale(built, [FAST_SOURCE]):
        return built
    import sysconfig

    import torch

    base = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    include = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], cuda]
    tmp = built + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{d}" for d in include), "-o", tmp,
           FAST_SOURCE, f"-L{os.path.join(base, 'lib')}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, built)
    return built


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the library if it is missing or older than its sources, then the Python module beside it; returns the
    library's path.  The module is optional (without it the attention operators' calls take the way through ctypes): a
    host that cannot compile it gets a warning."""
    if force or stale():
        tmp = LIB + ".tmp"
        cmd = [nvcc(), *NVCC_FLAGS, "-o", tmp, os.path.join(HERE, "csrc", "convrot.cu")]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB)
    try:
        build_fast(force, verbose)
    except (OSError, RuntimeError, ImportError, subprocess.CalledProcessError) as e:
        warnings.warn(f"the compiled calls of the attention operators were not built: {e}", RuntimeWarning, stacklevel=2)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))

"""Build memboost_b200/libmemboost_b200.so from memboost_b200/csrc/*.cu, and
memboost_b200/_calls.so from csrc/calls.cpp.

Every translation unit is compiled for sm_100a only
(-gencode arch=compute_100a,code=sm_100a) with -lineinfo, and linked into one
shared library with a statically linked CUDA runtime.  The library exports
exactly the C ABI declared in include/memboost_b200.h.  nvcc cross-compiles,
so this runs on machines without a GPU.  _calls.so is a CPython module over
torch's tensors that calls the library: it belongs to the torch and Python it was
built with, and is built again when either has changed.

Usage: python memboost_b200/build.py [--force] [-v]
(run by path: importing the package needs the library this builds)
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libmemboost_b200.so")
CALLS = os.path.join(PKG, "_calls.so")
CALLS_FOR = os.path.join(BUILD, "_calls.for")  # the torch and Python it was built with

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
              "--expt-relaxed-constexpr", "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else (shutil.which("nvcc") or "nvcc")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _headers():
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")))


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if _stale(obj, [src, __file__] + _headers()):
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        if verbose and r.stderr.strip():
            print(r.stderr, flush=True)
    return obj


def _torch() -> tuple[str, str]:
    """(directory, version) of the installed torch, without importing it."""
    where = importlib.util.find_spec("torch").submodule_search_locations[0]
    scope: dict = {}
    with open(os.path.join(where, "version.py")) as f:
        exec(f.read(), scope)
    return where, str(scope["__version__"])


def _calls_stale(made_for: str) -> bool:
    src = os.path.join(CSRC, "calls.cpp")
    if _stale(CALLS, [src, __file__, os.path.join(INCLUDE, "memboost_b200.h")]):
        return True
    if not os.path.exists(CALLS_FOR):
        return True
    with open(CALLS_FOR) as f:
        return f.read() != made_for


def _build_calls(verbose: bool) -> None:
    torch, version = _torch()
    made_for = f"torch {version}, Python {sysconfig.get_python_version()}\n"
    if not _calls_stale(made_for):
        return
    src = os.path.join(CSRC, "calls.cpp")
    system = [os.path.join(torch, "include"),
              os.path.join(torch, "include", "torch", "csrc", "api", "include"),
              sysconfig.get_paths()["include"],
              os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")]
    tmp = CALLS + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-I", INCLUDE,
           f'-DMB_TORCH_VERSION="{version}"']
    for d in system:
        cmd += ["-isystem", d]
    cmd += [src, "-o", tmp, "-L", PKG, "-l:libmemboost_b200.so", "-L", os.path.join(torch, "lib"),
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building {CALLS} failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, CALLS)
    with open(CALLS_FOR, "w") as f:
        f.write(made_for)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    if force:
        for o in glob.glob(os.path.join(BUILD, "*.o")):
            os.remove(o)
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if force or _stale(LIB, objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if force and os.path.exists(CALLS):
        os.remove(CALLS)
    _build_calls(verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

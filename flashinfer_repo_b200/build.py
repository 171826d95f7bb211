"""Build the C-ABI shared library libdsa_b200.so (sm_100a) in-tree.

    python -m flashinfer_repo_b200.build [--force]

Compiles every csrc/*.cu and csrc/step/*.cu with nvcc for sm_100a only, links the CUDA runtime
statically (so the library loads on machines without a driver, e.g. for the
symbol checks) and writes flashinfer_repo_b200/libdsa_b200.so.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libdsa_b200.so")
BUILD_DIR = os.path.join(PKG, "_build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-I", INCLUDE,
]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "step", "*.cu")))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD_DIR, exist_ok=True)
    headers = (glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "step", "*.cuh")) +
               glob.glob(os.path.join(INCLUDE, "*.h")))
    objs = []
    procs = []
    for src in sources():
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc()] + NVCC_FLAGS + ["-c", src, "-o", obj]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                                stderr=subprocess.STDOUT, text=True)))
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stderr.write(out)
        if p.returncode:
            raise RuntimeError(f"nvcc failed on {src}")
    if force or _stale(LIB, objs):
        cmd = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared",
               "-cudart", "static", "-o", LIB] + objs
        subprocess.check_call(cmd)
    return LIB


PROBES = os.path.join(PKG, "probes")


def build_probes(force: bool = False) -> list:
    """Compile the measurement probes in probes/*.cu (standalone programs, not
    part of the library) next to their sources."""
    outs = []
    for src in sorted(glob.glob(os.path.join(PROBES, "*.cu"))):
        exe = src[:-3]
        if force or _stale(exe, [src] + glob.glob(os.path.join(CSRC, "*.cuh")) +
                           glob.glob(os.path.join(CSRC, "step", "*.cuh"))):
            subprocess.check_call([nvcc()] + NVCC_FLAGS + ["-o", exe, src, "-lcuda"])
        outs.append(exe)
    return outs


def build_contest_binding(force: bool = False) -> str | None:
    """Compile the contest route's TVM-FFI binding (contest/binding.cu) for
    sm_100a into _build/ as a check that it builds; the contest harness itself
    compiles the packed sources with tvm_ffi.cpp.load.  Skipped (None) when
    tvm_ffi is not installed."""
    try:
        import tvm_ffi
    except ImportError:
        return None
    src = os.path.join(PKG, "contest", "binding.cu")
    obj = os.path.join(BUILD_DIR, "contest_binding.o")
    os.makedirs(BUILD_DIR, exist_ok=True)
    if force or _stale(obj, [src, os.path.join(INCLUDE, "dsa_b200.h")]):
        inc = os.path.join(os.path.dirname(tvm_ffi.__file__), "include")
        subprocess.check_call([nvcc()] + NVCC_FLAGS + ["-I", ROOT, "-I", inc, "-c", src, "-o", obj])
    return obj


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    if "--probes" in sys.argv:
        print("\n".join(build_probes(force="--force" in sys.argv)))

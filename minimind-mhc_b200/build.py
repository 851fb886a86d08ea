"""Build the sm_100a shared library ``model/libmhc_b200.so`` with nvcc.

The library is the C-ABI boundary declared in ``include/mhc_b200.h``; it links
only the CUDA runtime (no PyTorch headers), so any FFI can bind it.  Beside it
``model/_mhc_torch.so`` is compiled from ``csrc/host``: the PyTorch host side of
the training-step operators, which calls the library through its C header.  Objects go
to ``_build/`` at the repository root; every translation unit compiles in
parallel.  Usage::

    python minimind-mhc_b200/build.py [--force] [--ptxas-verbose]
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "model", "libmhc_b200.so")
HOST_LIB = os.path.join(PKG, "model", "_mhc_torch.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2",
          "--expt-relaxed-constexpr", f"-I{INCLUDE}", f"-I{CSRC}"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps():
    return [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))] + [
        os.path.join(INCLUDE, "mhc_b200.h")]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, ptxas_verbose: bool = False, quiet: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    nvcc = _nvcc()
    headers = [d for d in _deps() if not d.endswith(".cu")]
    objs, jobs = [], []
    for src in sources():
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc] + ARCH + CFLAGS + (["-Xptxas", "-v"] if ptxas_verbose else []) + ["-c", src, "-o", obj]
            jobs.append((src, cmd))

    def run(job):
        src, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        return src, r

    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            for src, r in ex.map(run, jobs):
                if r.returncode != 0:
                    sys.stderr.write(r.stdout + r.stderr)
                    raise RuntimeError(f"nvcc failed on {os.path.basename(src)}")
                if ptxas_verbose or (not quiet and r.stderr.strip()):
                    sys.stderr.write(r.stderr)
    if force or jobs or _stale(LIB, objs):
        cmd = [nvcc] + ARCH + ["-shared", "-o", LIB] + objs + ["-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    if not quiet:
        print(f"built {LIB}")
    return LIB


def build_host(force: bool = False, quiet: bool = False) -> str:
    """The PyTorch host module (a C++ compile against torch's headers, about a minute)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    src = os.path.join(CSRC, "host", "mhc_torch.cpp")
    if not force and not _stale(HOST_LIB, [src, os.path.join(INCLUDE, "mhc_b200.h")]):
        return HOST_LIB
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    incs = include_paths() + [os.path.join(cuda, "include"), INCLUDE, sysconfig.get_paths()["include"]]
    libs = library_paths()
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_mhc_torch",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-isystem{i}" for i in incs], src, "-o", HOST_LIB, *[f"-L{p}" for p in libs],
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed on mhc_torch.cpp")
    if not quiet:
        print(f"built {HOST_LIB}")
    return HOST_LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true")
    a = ap.parse_args()
    build(force=a.force, ptxas_verbose=a.ptxas_verbose)
    build_host(force=a.force)

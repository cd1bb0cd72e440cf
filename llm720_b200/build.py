"""Build the CUDA library in-tree: ``python -m llm720_b200.build``.

Every ``csrc/*.cu`` is compiled for sm_100a only and linked into
``llm720_b200/lib/libpeer_b200.so`` (a plain C-ABI shared object, no Python or
torch symbols).  Sources are compiled in parallel; an object is rebuilt only
when it is older than its source or any header.

``csrc/torch/row_ops.cpp``, the torch binding of the row-wise operators, becomes
``llm720_b200/lib/_row_ops.so``, a Python extension that links against the
library beside it.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "build")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libpeer_b200.so")
EXT = os.path.join(LIBDIR, "_row_ops.so")
EXT_SRC = os.path.join(CSRC, "torch", "row_ops.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _extension_command():
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ce
    includes = ce.include_paths("cuda") + [sysconfig.get_paths()["include"],
                                           os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_row_ops",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + [f"-I{p}" for p in includes]
            + [EXT_SRC, "-o", EXT] + [f"-L{p}" for p in ce.library_paths("cuda")]
            + [f"-L{LIBDIR}", "-lpeer_b200", "-Wl,-rpath,$ORIGIN", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
               "-ltorch_python"])


def build_extension(force: bool = False, verbose: bool = False) -> str:
    """The torch binding; rebuilt when its source, the C header or the installed torch is newer."""
    import torch
    deps = [EXT_SRC, os.path.join(os.path.dirname(PKG), "include", "peer_b200.h"), torch.version.__file__]
    if force or _stale(EXT, deps):
        r = subprocess.run(_extension_command(), capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(f"[{os.path.basename(EXT_SRC)}]\n{r.stdout}{r.stderr}")
        if r.returncode:
            raise RuntimeError(f"g++ failed on {EXT_SRC}")
    return EXT


def build_library(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    nvcc = _nvcc()
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = (glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh"))
               + glob.glob(os.path.join(os.path.dirname(PKG), "include", "*.h")))
    jobs = []
    for src in sources:
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info else []) + ["-c", src, "-o", obj]
            jobs.append((src, cmd))

    def run(job):
        src, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        return src, r

    with cf.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        for src, r in ex.map(run, jobs):
            if verbose or ptxas_info or r.returncode:
                sys.stderr.write(f"[{os.path.basename(src)}]\n{r.stdout}{r.stderr}")
            if r.returncode:
                raise RuntimeError(f"nvcc failed on {src}")
    objs = [os.path.join(OBJ, os.path.basename(s)[:-3] + ".o") for s in sources]
    if force or jobs or _stale(LIB, objs):
        cmd = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    build_extension(force, verbose)
    return LIB


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv))

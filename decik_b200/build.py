"""Build the native library ``decik_b200/lib/libdecik_b200.so`` from ``decik_b200/csrc/*.cu``.

Every source is compiled for sm_100a only (``-gencode arch=compute_100a,code=sm_100a``) with
nvcc, in parallel, into ``decik_b200/lib/obj/``, then linked into one shared library with the C ABI
declared in ``include/decik_b200.h``. A source is recompiled when it or any header under
``csrc/`` or ``include/`` is newer than its object. ``csrc/host/attn_inputs.cpp``, the torch binding of
the operators whose calls are short, becomes the CPython module ``decik_b200/lib/_attn_inputs.so``,
compiled by g++ against the installed torch and linked to the library beside it.

    python -m decik_b200.build [--force] [--verbose]
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIBDIR = os.path.join(PKG, "lib")
OBJDIR = os.path.join(LIBDIR, "obj")
LIB = os.path.join(LIBDIR, "libdecik_b200.so")
BIND_SRC = os.path.join(CSRC, "host", "attn_inputs.cpp")
BIND = os.path.join(LIBDIR, "_attn_inputs.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "include")]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found (set NVCC)")
    return cand


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, force: bool, verbose: bool, extra: list[str]) -> str:
    obj = os.path.join(OBJDIR, os.path.basename(src)[:-3] + ".o")
    if (not force and os.path.exists(obj)
            and os.path.getmtime(obj) >= max(os.path.getmtime(src), _headers_mtime())):
        return obj
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *extra, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr, flush=True)
    return obj


def _build_bind(force: bool, verbose: bool) -> None:
    import torch

    stamp = os.path.join(OBJDIR, "attn_inputs.torch")  # the torch it was built against
    built_for = open(stamp).read() if os.path.exists(stamp) else ""
    if (not force and os.path.exists(BIND) and built_for == torch.__version__
            and os.path.getmtime(BIND) >= max(os.path.getmtime(BIND_SRC), _headers_mtime())):
        return
    base = os.path.join(os.path.dirname(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DDECIK_TORCH_VERSION="{torch.__version__}"', "-I", os.path.join(ROOT, "include"),
           "-isystem", os.path.join(base, "include"), "-isystem", os.path.join(cuda, "include"),
           "-isystem", sysconfig.get_paths()["include"], BIND_SRC, "-o", BIND + ".tmp",
           "-L", LIBDIR, "-ldecik_b200", "-Wl,-rpath,$ORIGIN", "-L", os.path.join(base, "lib"), "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {os.path.basename(BIND_SRC)}:\n{res.stdout}\n{res.stderr}")
    os.replace(BIND + ".tmp", BIND)
    with open(stamp, "w") as f:
        f.write(torch.__version__)


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> str:
    os.makedirs(OBJDIR, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    extra = ["-Xptxas", "-v"] if ptxas_verbose else []
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force or ptxas_verbose, verbose or ptxas_verbose, extra), sources))
    if force or not os.path.exists(LIB) or max(os.path.getmtime(o) for o in objs) > os.path.getmtime(LIB):
        cmd = [nvcc(), *ARCH, "-shared", "-o", LIB + ".tmp", *objs, "-lcuda"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(LIB + ".tmp", LIB)
    _build_bind(force, verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas", action="store_true", help="print registers / spills / smem per kernel")
    a = ap.parse_args()
    print(build(a.force, a.verbose, a.ptxas))
    sys.exit(0)

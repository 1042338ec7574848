"""Build ``libqx_b200.so`` (the C-ABI library) from ``csrc/*.cu`` with nvcc.

    python -m qextract_infer_b200.build [--force] [--verbose] [--trace]

Compiles every ``.cu`` file for sm_100a only (``-gencode
arch=compute_100a,code=sm_100a``) into ``_build/*.o`` and links the shared
library next to this file, so it travels with the source tree.  Objects are
rebuilt when their source or any header is newer.

``--trace`` builds the profiling library ``libqx_b200_trace.so`` instead
(objects in ``_build_trace/``, compiled with ``-DQX_TRACE``): the same kernels
with per-CTA phase timestamps, recorded when ``qx_trace_launches`` is given a
buffer (``bench.py --workload timeline`` reads them).  The package never loads
it; the product library carries no trace code.

Beside the library it builds ``_binding.so`` from ``csrc/binding.cpp`` with g++
against torch's headers: the Python binding of the operators whose host side
counts (it calls the library's C ABI).
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libqx_b200.so")
BUILD_TRACE = os.path.join(PKG, "_build_trace")
LIB_TRACE = os.path.join(PKG, "libqx_b200_trace.so")
BINDING = os.path.join(PKG, "_binding.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found (CUDA toolkit required to build libqx_b200.so)")
    return cand


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _read(path):
    if not os.path.exists(path):
        return None
    with open(path) as f:
        return f.read()


def build(force: bool = False, verbose: bool = False, extra_flags=None, trace: bool = False) -> str:
    build_dir, lib = (BUILD_TRACE, LIB_TRACE) if trace else (BUILD, LIB)
    os.makedirs(build_dir, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdrs = _headers()
    flags = NVCC_FLAGS + list(extra_flags or []) + (["-DQX_TRACE"] if trace else [])
    nv = nvcc()

    def compile_one(src):
        obj = os.path.join(build_dir, os.path.basename(src)[:-3] + ".o")
        if force or _stale(obj, [src] + hdrs):
            cmd = [nv, *ARCH, *flags, "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
            if verbose and (r.stdout or r.stderr):
                print(r.stdout + r.stderr, flush=True)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, len(srcs) or 1)) as ex:
        objs = list(ex.map(compile_one, srcs))
    if force or _stale(lib, objs):
        tmp = lib + f".tmp{os.getpid()}"
        cmd = [nv, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, lib)
    if not trace:
        build_binding(force=force, verbose=verbose)
    return lib


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """``_binding.so``, linked against ``libqx_b200.so`` beside it and torch; rebuilt when
    torch or Python are others than those it was built with, too."""
    import sysconfig

    import torch
    src = os.path.join(CSRC, "binding.cpp")
    stamp = os.path.join(BUILD, "binding.stamp")
    made_for = (f"torch {torch.__version__} cuda {torch.version.cuda} cxx11abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} "
                f"python {sysconfig.get_config_var('SOABI')}\n")
    if not (force or _stale(BINDING, [src, os.path.join(INCLUDE, "qx_b200.h")]) or _read(stamp) != made_for):
        return BINDING
    from torch.utils import cpp_extension
    tmp = BINDING + f".tmp{os.getpid()}"
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include")]
    for d in cpp_extension.include_paths():
        cmd += ["-isystem", d]
    cmd += [src, "-o", tmp, "-L", PKG, "-l:libqx_b200.so", "-Wl,-rpath,$ORIGIN", "-L", lib, "-lc10", "-lc10_cuda",
            "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING)
    os.makedirs(BUILD, exist_ok=True)
    with open(stamp, "w") as f:
        f.write(made_for)
    return BINDING


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--trace", action="store_true", help="build the profiling library libqx_b200_trace.so")
    a = ap.parse_args(argv)
    print(build(force=a.force, verbose=a.verbose, trace=a.trace))


if __name__ == "__main__":
    main(sys.argv[1:])

"""Build libgrouped_gemm_b200.so in place (sm_100a only).

    python -m grouped_gemm_gpu_kernel_b200.build [--verbose]

Compiles every CUDA / C++ source under csrc/ with nvcc for ``arch=compute_100a,code=sm_100a``
and links one shared library next to this file. The static CUDA runtime is linked in, so the
library needs only the driver at run time; it is loaded with ctypes (Python) or linked directly
(C/C++ callers of include/grouped_gemm_b200.h or include/grouped_gemm/grouped_gemm.cuh). On top of it
csrc/moe_python.cpp becomes _moe_native.<ABI>.so, a CPython module that only the package's
mixture-of-experts calls use (g++ and Python.h); where those are missing the library is all that is
made, and these calls raise.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_NAME = "libgrouped_gemm_b200.so"
LIB_PATH = os.path.join(PKG, LIB_NAME)
# the Python calls of the mixture-of-experts operators, named for the interpreter that they are compiled for
CALLS_PATH = os.path.join(PKG, "_moe_native" + sysconfig.get_config_var("EXT_SUFFIX"))
BUILD_DIR = os.path.join(PKG, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr", "-I" + INCLUDE, "-I" + CSRC]
SOURCES = ["gg_kernels.cu", "gg_host.cu", "gg_copy.cu", "gg_simt.cu", "gg_ipc.cu", "gg_router.cu",
           "gg_rows.cu", "gg_q4.cu", "grouped_gemm_api.cpp"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise FileNotFoundError("nvcc not found")


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"command failed ({res.returncode}): {' '.join(cmd[:3])} ...")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr)
    return res


def _newer(target: str, deps) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


CALLS_SOURCE = os.path.join(CSRC, "moe_python.cpp")


def _deps():
    out = []
    for root in (CSRC, INCLUDE):
        for dirpath, _, files in os.walk(root):
            out += [os.path.join(dirpath, f) for f in files if f.endswith((".cu", ".cuh", ".h", ".cpp"))]
    out.remove(CALLS_SOURCE)
    return out


def build(verbose: bool = False, force: bool = False, ptxas_info: bool = False) -> str:
    if force or ptxas_info or not _newer(LIB_PATH, _deps() + [__file__]):
        _build_library(verbose, ptxas_info)
    if force or not _newer(CALLS_PATH, [CALLS_SOURCE, os.path.join(INCLUDE, "grouped_gemm_b200.h"), __file__]):
        _build_calls(verbose)
    return LIB_PATH


def _build_library(verbose: bool, ptxas_info: bool) -> None:
    os.makedirs(BUILD_DIR, exist_ok=True)
    cc = nvcc()
    objs = [os.path.join(BUILD_DIR, os.path.splitext(src)[0] + ".o") for src in SOURCES]

    def compile_one(src, obj):
        extra = ["-Xptxas", "-v"] if (ptxas_info and src.endswith(".cu")) else []
        lang = ["-x", "cu"] if src.endswith(".cu") else []
        return _run([cc, *ARCH, *NVCC_FLAGS, *extra, *lang, "-c", os.path.join(CSRC, src), "-o", obj], verbose)

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as pool:
        for res in pool.map(compile_one, SOURCES, objs):
            if ptxas_info:
                sys.stdout.write(res.stderr)
    tmp = LIB_PATH + ".tmp"
    _run([cc, *ARCH, "-shared", "-o", tmp, *objs, "-lcudart_static", "-ldl", "-lrt", "-lpthread"], verbose)
    os.replace(tmp, LIB_PATH)


def _build_calls(verbose: bool) -> None:
    """The CPython module on top of the library, which it finds beside itself. The library's other callers do not need
    it, so its absence is a warning."""
    cxx, headers = shutil.which("g++"), sysconfig.get_paths()["include"]
    if not cxx or not os.path.exists(os.path.join(headers, "Python.h")):
        if os.path.exists(CALLS_PATH):
            os.remove(CALLS_PATH)  # of other sources than the library's
        warnings.warn(f"{os.path.basename(CALLS_PATH)} was not built: " +
                      (f"no Python.h in {headers}" if cxx else "no g++") +
                      "; the package's mixture-of-experts calls will raise")
        return
    tmp = CALLS_PATH + ".tmp"
    _run([cxx, "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-I" + INCLUDE, "-I" + headers, CALLS_SOURCE, "-o", tmp,
          "-L" + PKG, "-l:" + LIB_NAME, "-Wl,-rpath,$ORIGIN"], verbose)
    os.replace(tmp, CALLS_PATH)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print -Xptxas -v register/smem usage")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force, ptxas_info=a.ptxas_info))


if __name__ == "__main__":
    main()

"""Build libneurodsl_b200.so in-tree with nvcc for sm_100a.

    python -m neurodsl_b200.build [--force] [--verbose]

Each .cu under csrc/ is compiled separately (-gencode arch=compute_100a,
code=sm_100a, -O3, -lineinfo) and linked into neurodsl_b200/libneurodsl_b200.so
with the CUDA runtime linked statically, so the library only needs the driver
at load time.  No GPU is needed to build.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import warnings

from . import _lib

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libneurodsl_b200.so")
SOURCES = ["abi.cu", "tma.cu", "flash_fwd.cu", "kv_decode.cu", "gemm.cu", "layernorm.cu", "model_ops.cu",
           "tp_comm.cu", "elementwise.cu", "paged_decode.cu", "paged_kv.cu", "logits.cu"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-fvisibility=hidden", "-I", os.path.join(ROOT, "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or install the CUDA toolkit)")


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    return hs + [os.path.join(ROOT, "include", "neurodsl_b200.h")]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False, extra_flags=None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    cc = nvcc()
    headers = _headers()
    flags = NVCC_FLAGS + list(extra_flags or [])
    jobs = []
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmd = [cc] + ARCH + flags + ["-c", s, "-o", o]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    failed = []
    with cf.ThreadPoolExecutor(max_workers=min(8, len(jobs) or 1)) as ex:
        for cmd, r in ex.map(run, jobs):
            if verbose or r.returncode != 0:
                sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
            if r.returncode != 0:
                failed.append(cmd[-3])
    if failed:
        raise RuntimeError(f"nvcc failed for: {failed}")
    if force or jobs or _stale(LIB, objs):
        cmd = [cc] + ARCH + ["-shared", "-o", LIB] + objs + ["-Xcompiler", "-fPIC"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    return LIB


def build_calls(force: bool = False):
    """neurodsl_b200/_calls.<interpreter>.<torch>.so: the CPython extension that
    makes the serving operators' calls (csrc/py_calls.cpp), against this interpreter
    and its torch.  None, with a warning, where there is no torch, no C++ compiler or
    none of their headers: ctypes then makes the calls."""
    import sysconfig
    try:
        import torch
        from torch.utils.cpp_extension import include_paths
    except ImportError as e:
        return _no_calls(e)
    target = _lib.calls_path()
    src = os.path.join(CSRC, "py_calls.cpp")
    if not force and not _stale(target, [src, os.path.join(ROOT, "include", "neurodsl_b200.h")]):
        return target
    cxx = os.environ.get("CXX", "g++")
    if shutil.which(cxx) is None:
        return _no_calls(f"no C++ compiler ({cxx})")
    for header, dirs in (("Python.h", [sysconfig.get_paths()["include"]]),
                         ("torch/csrc/autograd/python_variable.h", include_paths())):
        if not any(os.path.exists(os.path.join(d, header)) for d in dirs):
            return _no_calls(f"no {header}")
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", os.path.join(ROOT, "include"), "-isystem", sysconfig.get_paths()["include"],
           "-isystem", os.path.join(cuda, "include")]
    for d in include_paths():
        cmd += ["-isystem", d]
    cmd += [src, "-o", target, "-L", libs, "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("building the calls' extension failed:\n" + r.stdout + r.stderr)
    return target


def _no_calls(why):
    warnings.warn(f"the calls' extension is not built: {why}", stacklevel=3)
    return None


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
    print(build_calls(force=a.force))


if __name__ == "__main__":
    main()

"""Build libchronoquant_b200.so in-tree with nvcc for sm_100a.

    python -m chronoquant_mlx_b200.build [--force] [-j N] [--checks]

Each ``csrc/*.cu`` compiles to an object under ``_build/`` (in parallel), then
they link into ``chronoquant_mlx_b200/libchronoquant_b200.so``.  Objects are
rebuilt when their source or any ``csrc/*.cuh`` / ``include/*.h`` is newer.
``csrc/cq_calls.cpp`` (host code: the checked Python entry points of the sparse
operators) compiles with g++ against torch's headers into the extension module
``chronoquant_mlx_b200/_calls.so``.

``--checks`` builds the debug variant ``libchronoquant_b200_checks.so``
(objects under ``_build/checks/``) with ``-DCQ_CHECKS``: every page lookup
in the kernels is bounds-checked and a bad index is reported as device
error 7 (``cq_device_error``) instead of being followed.  The package loads
it instead of the release library when ``CQ_CHECKS=1`` is set at import.
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libchronoquant_b200.so")
OUT_CHECKS = os.path.join(HERE, "libchronoquant_b200_checks.so")
BUILD = os.path.join(ROOT, "_build")
CALLS_SRC = os.path.join(CSRC, "cq_calls.cpp")
CALLS_OUT = os.path.join(HERE, "_calls.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", os.path.join(ROOT, "include"), "-I", CSRC]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _newest_header() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def build_calls(force: bool = False) -> str:
    """The extension module of cq_calls.cpp (rebuilt when it, the C header or torch's version is newer)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    stamp = os.path.join(BUILD, "calls.torch")
    header = os.path.join(ROOT, "include", "chronoquant_b200.h")
    version = f"{torch.__version__} {sysconfig.get_python_version()}"
    built_for = open(stamp).read() if os.path.exists(stamp) else ""
    if (not force and built_for == version and os.path.exists(CALLS_OUT)
            and os.path.getmtime(CALLS_OUT) >= max(os.path.getmtime(CALLS_SRC), os.path.getmtime(header))):
        return CALLS_OUT
    os.makedirs(BUILD, exist_ok=True)
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    inc = [f for d in (*cpp_extension.include_paths(), cuda, sysconfig.get_paths()["include"]) for f in ("-isystem", d)]
    tmp = CALLS_OUT + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *inc, CALLS_SRC, "-o", tmp, "-L", lib,
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {CALLS_SRC}:\n{r.stderr}")
    os.replace(tmp, CALLS_OUT)
    with open(stamp, "w") as f:
        f.write(version)
    return CALLS_OUT


def build(force: bool = False, jobs: int = 8, verbose: bool = False, checks: bool = False) -> str:
    bdir = os.path.join(BUILD, "checks") if checks else BUILD
    out = OUT_CHECKS if checks else OUT
    os.makedirs(bdir, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr = _newest_header()
    cc = nvcc()
    flags = FLAGS + (["-DCQ_CHECKS"] if checks else [])

    def compile_one(src: str) -> str:
        obj = os.path.join(bdir, os.path.basename(src)[:-3] + ".o")
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr):
            return obj
        cmd = [cc, *ARCH, *flags, "-Xptxas", "-v", "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
        if verbose:
            sys.stderr.write(r.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=jobs) as ex:
        calls = ex.submit(build_calls, force)
        objs = list(ex.map(compile_one, srcs))
    newest_obj = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(out) or os.path.getmtime(out) < newest_obj:
        tmp = out + ".tmp"
        cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
        os.replace(tmp, out)
    calls.result()  # reported once the library stands: a binding of the C ABI needs no extension
    return out


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=8)
    ap.add_argument("-v", action="store_true")
    ap.add_argument("--checks", action="store_true", help="the bounds-checked debug variant")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.j, verbose=a.v, checks=a.checks))


if __name__ == "__main__":
    main()

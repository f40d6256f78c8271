"""Build libmoe_b200.so (the C-ABI library) in-tree with nvcc for sm_100a, and _calls.so (the
dense operators' calls from Python) with g++ against torch's headers. The second is optional:
without it those calls go through ctypes, with the same results.

Usage: python mlx-rs_b200/build.py [--force] [--verbose]
Objects go to mlx-rs_b200/_build/, the libraries to mlx-rs_b200/.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libmoe_b200.so")
CALLS = os.path.join(HERE, "_calls.so")
CALLS_FOR = os.path.join(BUILD, "calls.for")  # what it was built against
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
                     "--expt-relaxed-constexpr", "-I" + CSRC, "-I" + INCLUDE]


def nvcc() -> str:
    p = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(p):
        raise RuntimeError("nvcc not found")
    return p


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False, extra_flags=None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    hdrs = headers()
    objs, jobs = [], []
    for src in sources():
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + hdrs):
            cmd = [nvcc()] + NVCC_FLAGS + (extra_flags or []) + ["-c", src, "-o", obj]
            jobs.append(cmd)

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"build failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, flush=True)

    with ThreadPoolExecutor(max_workers=max(1, min(8, os.cpu_count() or 1))) as ex:
        list(ex.map(run, jobs))
    if force or jobs or _stale(LIB, objs):
        cmd = [nvcc()] + ARCH + ["-shared", "-o", LIB] + objs + ["-lcudart"]
        run(cmd)
    src = os.path.join(CSRC, "torch_calls.cpp")
    try:
        if force or _stale(CALLS, [src] + [h for h in hdrs if h.startswith(INCLUDE)]) or _built_for() != calls_for():
            run(calls_command(src))
            with open(CALLS_FOR, "w") as f:
                f.write(calls_for())
    except (RuntimeError, OSError, ImportError) as e:  # no compiler, no headers of torch, no torch
        if os.path.exists(CALLS):
            os.remove(CALLS)  # it may not fit the library
        print(f"{os.path.basename(CALLS)} was not built, the calls go through ctypes: {e}", file=sys.stderr)
    return LIB


def calls_for() -> str:
    """What _calls.so is built against."""
    import torch
    return f"{torch.__version__} {os.path.dirname(os.path.abspath(torch.__file__))} {sys.version}"


def _built_for():
    try:
        with open(CALLS_FOR) as f:
            return f.read()
    except OSError:
        return None


def calls_command(src: str):
    import sysconfig

    import torch
    troot = os.path.dirname(os.path.abspath(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    inc = [os.path.join(troot, "include"), os.path.join(troot, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    return ["g++", "-O2", "-fPIC", "-shared", "-std=c++17", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[f"-I{d}" for d in inc], src, "-o", CALLS, f"-L{HERE}", "-l:libmoe_b200.so", f"-L{os.path.join(troot, 'lib')}",
            "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)

"""Build kyro_b200/libkyro_spec.so from kyro_b200/csrc/*.cu with nvcc for sm_100a.

Usage: python -m kyro_b200.build [--force] [--verbose]

Each translation unit compiles to an object under kyro_b200/_build/, then
nvcc links them into one shared library with the CUDA runtime linked
statically (the library exports only the C ABI of include/kyro_spec.h).
csrc/pycall.cpp, the Python calls of the chunk operators, becomes an extension
module beside it, for the torch and the Python that it is built with: it reads
torch's tensors in place, so its file is named after both (pycall_path).
Without torch's or Python's headers, or a host C++ compiler, the library is
built all the same.
sampler.cu is compiled with --fmad=false: its arithmetic must round exactly
like the CPU restatement it is checked against.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libkyro_spec.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-ffp-contract=off",
          "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]
PER_FILE = {"sampler.cu": ["--fmad=false"]}


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def headers():
    return [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))] + [
        os.path.join(ROOT, "include", "kyro_spec.h")]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    cc = nvcc()
    hdrs = headers()
    objs = []
    for src in sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src[:-3] + ".o")
        objs.append(o)
        if force or _stale(o, [s] + hdrs + [__file__]):
            cmd = [cc, *ARCH, *COMMON, *PER_FILE.get(src, []), "-c", s, "-o", o]
            if verbose:
                cmd += ["-Xptxas", "-v"]
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
    if force or _stale(LIB, objs):
        cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs, "-ldl", "-lpthread"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    _build_pycall(force, verbose)
    return LIB


def pycall_path(torch_version: str) -> str:
    """The extension module for this Python and a version of torch."""
    return os.path.join(HERE, f"_pycall-torch{torch_version}"
                        f"{sysconfig.get_config_var('EXT_SUFFIX')}")


def _build_pycall(force: bool, verbose: bool):
    src = os.path.join(CSRC, "pycall.cpp")
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return _no_pycall("torch is not installed")
    torch = os.path.dirname(spec.origin)
    out = pycall_path(runpy.run_path(os.path.join(torch, "version.py"))["__version__"])
    if not (force or _stale(out, [src, os.path.join(ROOT, "include", "kyro_spec.h"), __file__])):
        return
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    inc = [os.path.join(torch, "include"),
           os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include"),
           os.path.join(ROOT, "include")]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           *["-I" + i for i in inc], src, "-o", out, "-L" + os.path.join(torch, "lib"),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    if os.path.exists(out):
        os.remove(out)
    try:
        subprocess.run(cmd, check=True)
    except (OSError, subprocess.CalledProcessError) as e:
        _no_pycall(str(e))


def _no_pycall(why: str):
    """The library is complete without the module; its calls are what it is for."""
    print(f"kyro_b200: no extension module, Python calls go through ctypes ({why})",
          file=sys.stderr, flush=True)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args(argv)
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    sys.exit(main())

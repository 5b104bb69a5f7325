"""Build the sm_100a sampler library in-tree.

    python -m noel_b200.build          # generate the expf table, compile the .so

Steps:
1. ``csrc/gen_expf_table.cc`` (host C++, OpenMP) lists the inputs of (-15, 0]
   where the C library's expf differs from the correctly rounded exp, into
   ``csrc/_gen/expf_table.inc``.  It calls the C library's expf on this host,
   so the table matches the libm the reference sampler links against.
2. nvcc compiles the units of ``csrc`` for sm_100a side by side and links them
   into ``noel_b200/libnoel_sampler_cuda.so`` (C ABI of include/).
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
GEN = os.path.join(CSRC, "_gen")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libnoel_sampler_cuda.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    *ARCH, "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-warn-spills",
]
# the library's translation units, and the headers of csrc that the smaller ones take
UNITS = {"sampler_cuda": None, "int8": ("host.h", "int8.cuh"), "requests": ("host.h", "requests.cuh")}


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _run(cmd, **kw):
    r = subprocess.run(cmd, capture_output=True, text=True, **kw)
    if r.returncode != 0:
        raise RuntimeError(f"command failed ({r.returncode}): {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return r


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def gen_table(force: bool = False) -> str:
    os.makedirs(GEN, exist_ok=True)
    src = os.path.join(CSRC, "gen_expf_table.cc")
    exe = os.path.join(GEN, "gen_expf_table")
    inc = os.path.join(GEN, "expf_table.inc")
    deps = [src, os.path.join(CSRC, "ref_expf.h")]
    if force or _stale(exe, deps):
        _run(["g++", "-O2", "-std=c++17", "-fopenmp", "-ffp-contract=off", src, "-o", exe, "-lm"])
    if force or _stale(inc, [exe]):
        _run([exe, inc, os.path.join(GEN, "expf_table.bin")])
    return inc


def build(force: bool = False, verbose: bool = False) -> str:
    inc = gen_table(force)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))]
    deps += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)] + [inc]
    if force or _stale(LIB, deps):
        headers = [d for d in deps if not d.endswith(".cu")]

        def compile(name):
            src, obj = os.path.join(CSRC, name + ".cu"), os.path.join(GEN, name + ".o")
            # a unit's own kernels and what it shares with others: the sampler's headers are not the other units'
            own = headers if name == "sampler_cuda" else [h for h in headers if os.path.basename(h) in UNITS[name]
                                                          or os.path.dirname(h) == INCLUDE]
            if not force and not _stale(obj, [src, *own]):
                return obj, ""
            cmd = [_nvcc(), *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj + ".tmp"]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            r = _run(cmd)
            os.replace(obj + ".tmp", obj)
            return obj, r.stderr

        with concurrent.futures.ThreadPoolExecutor() as pool:
            done = list(pool.map(compile, UNITS))
        _run([_nvcc(), *ARCH, "-shared", *[obj for obj, _ in done], "-o", LIB + ".tmp"])
        os.replace(LIB + ".tmp", LIB)
        if verbose:
            print("".join(err for _, err in done))
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

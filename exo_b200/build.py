"""Builds the CUDA library in-tree: exo_b200/libexo_b200.so (sm_100a only).

    python -m exo_b200.build [--force] [--verbose]

Each .cu under exo_b200/csrc is compiled with
``nvcc -gencode arch=compute_100a,code=sm_100a -lineinfo`` (the arch-specific
target: tcgen05 does not assemble for plain sm_100) and linked with the static
CUDA runtime, so the shared object depends on nothing but libstdc++ and the
driver.  nvcc cross-compiles without a GPU present.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(HERE, "libexo_b200.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
# the tag keeps another interpreter from importing it
CALL = os.path.join(HERE, "_call" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-fvisibility=hidden", "-I", INCLUDE,
]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    hs.append(os.path.join(INCLUDE, "exo_b200.h"))
    return hs


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(OBJ, exist_ok=True)
    headers = _headers()
    jobs = []
    objs = []
    for src in _sources():
        path = os.path.join(CSRC, src)
        obj = os.path.join(OBJ, src[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [path, *headers]):
            cmd = [nvcc, *NVCC_FLAGS, "-c", path, "-o", obj]
            if verbose:
                cmd[1:1] = ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    with concurrent.futures.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        for cmd, r in ex.map(run, jobs):
            if verbose or r.returncode != 0:
                sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed for {cmd[-3]}")
    if force or jobs or _stale(LIB, objs):
        cmd = [nvcc, "-shared", "-o", LIB, *objs, "-cudart", "static",
               "-gencode", "arch=compute_100a,code=sm_100a"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    build_call(force)
    return LIB


def _remove(path):
    try:
        os.remove(path)
    except FileNotFoundError:
        pass


def build_call(force: bool = False) -> "str | None":
    """The Python binding's fast path (csrc/call.cpp), a plain CPython module.  The package works without it, only
    slower by a few microseconds a call, so an interpreter without its headers or a machine without a C++ compiler is
    no error.  What it checks has to be what this source says: modules of an older source, and ones without an
    interpreter's tag, are removed whether or not a new one can be built."""
    src = os.path.join(CSRC, "call.cpp")
    for name in os.listdir(os.path.dirname(CALL)):
        path = os.path.join(os.path.dirname(CALL), name)
        if name == "_call.so" or (name.startswith("_call.") and name.endswith(".so") and _stale(path, [src])):
            _remove(path)
    if not force and os.path.exists(CALL):
        return CALL

    def without(why):
        sys.stderr.write(f"exo_b200: the binding's fast path is not built ({why})\n")

    headers = sysconfig.get_paths()["include"]
    if not os.path.exists(os.path.join(headers, "Python.h")):
        return without(f"no Python.h in {headers}")
    new = f"{CALL}.{os.getpid()}"  # a process may have the old one loaded
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-I", headers,
           src, "-o", new]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        return without(str(e))
    if r.returncode != 0:
        _remove(new)
        return without(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    os.replace(new, CALL)
    return CALL


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))

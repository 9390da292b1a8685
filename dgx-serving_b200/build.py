"""Builds libw4a8_b200.so (the C-ABI library) in-tree with nvcc for sm_100a.

Usage: python dgx-serving_b200/build.py [--force]
nvcc cross-compiles without a GPU; the explicit -gencode form is required because the tcgen05 / TMA
instructions exist only for the arch-specific target sm_100a.
"""
import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
SRCS = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".cu")]   # one object each, compiled side by side
OUT = os.path.join(HERE, "libw4a8_b200.so")
OBJ = os.path.join(HERE, "build")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ARCH + ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden"]


def sources():
    files = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC))]
    files.append(os.path.join(HERE, "..", "include", "w4a8_b200.h"))
    return files


def includes(path, seen=None):
    """`path` and what it includes by quoted name, recursively."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M):
                includes(os.path.join(os.path.dirname(path), name), seen)
    return seen


def up_to_date():
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(f) <= t for f in sources())


def compile_one(src, force, verbose):
    obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
    if not force and os.path.exists(obj) and all(os.path.getmtime(f) <= os.path.getmtime(obj) for f in includes(src)):
        return obj
    cmd = [NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", obj, src]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    if verbose:
        print(r.stderr)
    return obj


def build(force=False, verbose=False):
    """Compile the library unless it is newer than every source.  Returns the path of the .so."""
    if not force and up_to_date():
        return OUT
    if not os.path.exists(NVCC):
        if os.path.exists(OUT):
            return OUT  # no compiler here (a GPU box): use the prebuilt library that travelled with the tree
        raise RuntimeError("nvcc not found at %s and no prebuilt %s" % (NVCC, OUT))
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(len(SRCS)) as pool:
        objs = list(pool.map(lambda s: compile_one(s, force, verbose), SRCS))
    r = subprocess.run([NVCC] + ARCH + ["-shared", "-o", OUT] + objs, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

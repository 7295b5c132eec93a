"""Build ``chia_proj_b200/_lib/libchia_attn.so`` in-tree with nvcc for sm_100a.

    python -m chia_proj_b200.build [--force] [--verbose]

The library is a plain shared object with C linkage (``include/chia_attn.h``,
``include/chia_paged.h``);
it links the CUDA runtime statically and fetches ``cuTensorMapEncodeTiled``
from the driver at run time, so it needs no libcuda at link time. Beside it
stands a small CPython module (``csrc/binding.cpp``) that checks the tensors of
the paged cache's operators.
"""

from __future__ import annotations

import argparse
import glob
import importlib.metadata
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "_lib", "libchia_attn.so")
OBJ = os.path.join(HERE, "_lib", "_build")
# the binding is compiled against one torch version and named after it
BINDING_SRC = os.path.join(CSRC, "binding.cpp")
BINDING = os.path.join(HERE, "_lib", f"_binding-{importlib.metadata.version('torch')}.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-cudart", "static",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return sources() + sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + sorted(
        glob.glob(os.path.join(ROOT, "include", "*.h")))


def up_to_date() -> bool:
    if not os.path.exists(OUT) or not _binding_up_to_date():
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(d) <= t for d in _deps())


def _binding_up_to_date() -> bool:
    newest = max(os.path.getmtime(p) for p in (BINDING_SRC, *_headers(BINDING_SRC)))
    return os.path.exists(BINDING) and os.path.getmtime(BINDING) >= newest


def _build_binding(force: bool) -> None:
    """The CPython module over torch's C++ tensors (g++; no device code)."""
    if not force and _binding_up_to_date():
        return
    torch = os.path.dirname(importlib.util.find_spec("torch").origin)
    inc, lib = os.path.join(torch, "include"), os.path.join(torch, "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", "-D_GLIBCXX_USE_CXX11_ABI=1", "-o", BINDING + ".tmp", BINDING_SRC,
           "-isystem", inc, "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"),
           "-isystem", cuda, "-I", sysconfig.get_paths()["include"], "-L", lib, "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    subprocess.run(cmd, check=True)
    os.replace(BINDING + ".tmp", BINDING)


def _headers(src: str, seen=None):
    """The headers of this repository that ``src`` includes, directly or not."""
    seen = set() if seen is None else seen
    with open(src) as f:
        names = re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M)
    for n in names:
        p = os.path.normpath(os.path.join(os.path.dirname(src), n))
        if os.path.exists(p) and p not in seen:
            seen.add(p)
            _headers(p, seen)
    return seen


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if any source is newer; returns its path. Each
    source file is an object of its own, compiled only when it or one of its
    headers changed, several at a time."""
    if not force and up_to_date():
        return OUT
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJ, os.path.basename(src) + ".o")
        newest = max(os.path.getmtime(p) for p in (src, *_headers(src)))
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest:
            return obj
        cmd = [nvcc, *NVCC_FLAGS, "-c", "-I", os.path.join(ROOT, "include"), "-o", obj + ".tmp", src]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(obj + ".tmp", obj)
        return obj

    with ThreadPoolExecutor((os.cpu_count() or 1) + 1) as pool:
        binding = pool.submit(_build_binding, force)
        objects = list(pool.map(compile_one, sources()))
        binding.result()
    tmp = OUT + ".tmp"
    subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", tmp, *objects], check=True)
    os.replace(tmp, OUT)
    return OUT


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(force=a.force, verbose=a.verbose))


if __name__ == "__main__":
    sys.exit(main())

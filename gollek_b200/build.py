"""Builds libgollek_kernels.so (sm_100a) in-tree with nvcc.

    python -m gollek_b200.build            # build if sources changed
    python -m gollek_b200.build --force -v # rebuild, print ptxas register/spill report
"""
from __future__ import annotations

import argparse
import fcntl
import glob
import os
import shutil
import subprocess
import sys
import time
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libgollek_kernels.so")
HEADER = os.path.join(ROOT, "include", "gollek_kernels.h")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))) + [HEADER]


def stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(s) > t for s in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds the library if its sources are newer (or `force`).  Safe to call from several
    processes at once (the ranks of one job): one builds under an exclusive file lock while
    the others wait, then find it fresh; the new file replaces the old one atomically."""
    if not force and not stale():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    with open(os.path.join(LIB_DIR, ".build.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        if not force and not stale():
            return LIB_PATH
        return _build_locked(verbose)


def _build_locked(verbose: bool) -> str:
    tmp = f"{LIB_PATH}.{os.getpid()}.tmp"
    units = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    objs = [os.path.join(LIB_DIR, f"{os.path.basename(u)}.{os.getpid()}.o") for u in units]
    # The output carries the build's start time, so a source edited while nvcc runs still
    # reads as newer than the library.
    start = time.time()
    nvcc = [nvcc_path()]
    # nvcc's host compiler: prefer the system g++ (the environment's CXX may lack libgomp
    # or differ from what libstdc++ on the GPU box expects).
    if os.path.exists("/usr/bin/g++"):
        nvcc += ["-ccbin", "/usr/bin/g++"]
    flags = [*ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
             "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
             "-I", os.path.join(ROOT, "include")]
    if verbose:
        flags.append("-Xptxas=-v")

    def run(cmd):
        return subprocess.run(cmd, env=dict(os.environ), capture_output=True, text=True)

    try:
        # the translation units compile side by side, then link
        with ThreadPoolExecutor(len(units)) as pool:
            done = list(pool.map(lambda uo: run([*nvcc, *flags, "-c", "-o", uo[1], uo[0]]),
                                 zip(units, objs)))
        if all(r.returncode == 0 for r in done):
            done.append(run([*nvcc, *ARCH_FLAGS, "-shared", "-o", tmp, *objs]))
    finally:
        for o in objs:
            if os.path.exists(o):
                os.remove(o)
    if any(r.returncode != 0 for r in done):
        if os.path.exists(tmp):
            os.remove(tmp)
        sys.stderr.write("".join(r.stdout + r.stderr for r in done))
        raise RuntimeError("nvcc failed building libgollek_kernels.so")
    if verbose:
        sys.stderr.write("".join(r.stderr for r in done))
    os.utime(tmp, (start, start))
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))

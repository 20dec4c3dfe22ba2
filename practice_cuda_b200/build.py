"""Build libpcb200.so in-tree with nvcc for sm_100a.

``python -m practice_cuda_b200.build [--force]``.  The library is rebuilt
when any source under ``csrc/`` or ``include/`` is newer than it; each
``csrc/*.cu`` is compiled on its own, the out-of-date ones side by side.
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OUT = os.path.join(HERE, "_lib", "libpcb200.so")
PROF_OUT = os.path.join(HERE, "_lib", "libpcb200_prof.so")

NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler", "-fPIC",
]


def _sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*")) + glob.glob(os.path.join(ROOT, "include", "*.h")))


def needs_build(path: str = OUT) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(s) > t for s in _sources())


def _object_stale(obj: str) -> bool:
    """Whether a file that the object was compiled from (its ``.d`` list) is newer, or unknown."""
    if not os.path.exists(obj) or not os.path.exists(obj + ".d"):
        return True
    with open(obj + ".d") as f:
        deps = f.read().replace("\\\n", " ").split(":", 1)[-1].split()
    t = os.path.getmtime(obj)
    return any(not os.path.exists(d) or os.path.getmtime(d) > t for d in deps)


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libpcb200")
    return path


def build(force: bool = False, verbose: bool = False, profiling: bool = False, out: str | None = None) -> str:
    """Build the library.  ``profiling`` compiles the PCB200_PROFILING
    switches in (environment knobs that change kernel selection or skip work;
    never shipped) into ``out`` (default ``_lib/libpcb200_prof.so``)."""
    dst = out or (PROF_OUT if profiling else OUT)
    if not force and not needs_build(dst):
        return dst
    obj_dir = os.path.join(os.path.dirname(OUT), "obj_prof" if profiling else "obj")
    os.makedirs(obj_dir, exist_ok=True)
    os.makedirs(os.path.dirname(dst), exist_ok=True)
    objects, running = [], []
    for src in sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu"))):
        obj = os.path.join(obj_dir, os.path.basename(src) + ".o")
        objects.append(obj)
        if not force and not _object_stale(obj):
            continue
        cmd = [nvcc(), *NVCC_FLAGS, *(["-DPCB200_PROFILING"] if profiling else []), "-c", "-MMD", "-MF", obj + ".d",
               "-o", obj, src]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), file=sys.stderr)
        running.append((cmd, obj, subprocess.Popen(cmd)))
    failed = [(cmd, obj, p.returncode) for cmd, obj, p in running if p.wait() != 0]
    for _, obj, _ in failed:  # nvcc may leave a partial object behind
        if os.path.exists(obj):
            os.remove(obj)
    if failed:
        raise subprocess.CalledProcessError(failed[0][2], failed[0][0])
    tmp = dst + ".tmp"
    subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-o", tmp, *objects], check=True)
    os.replace(tmp, dst)
    return dst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--profiling", action="store_true", help="build libpcb200_prof.so with -DPCB200_PROFILING")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose, profiling=args.profiling))

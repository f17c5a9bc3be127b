"""Ahead-of-time build of the native library for sm_100a.

Produces ``tensorcore_gemm/_lib/libb200gemm.so`` next to the Python package,
in-tree, so a snapshot of the repository carries the built library with it.
The reference JIT-compiled its kernels on first call with load_inline and an
arch taken from whatever GPU was present (tensorcore_gemm/cuda_compile.py:47-62,
157-269); this library is compiled once, explicitly for sm_100a, and needs no
GPU to build.

Usage:  python ampere-gemm_b200/build.py [--force] [--verbose]
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
import tempfile
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
LIB_DIR = PKG_ROOT / "tensorcore_gemm" / "_lib"
LIB_PATH = LIB_DIR / "libb200gemm.so"
HEADERS = [REPO_ROOT / "include" / "b200_gemm.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xptxas", "-v",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; the B200 GEMM library cannot be built")


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + HEADERS


def needs_build() -> bool:
    if not LIB_PATH.exists():
        return True
    t = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > t for p in _sources())


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every csrc/*.cu (in parallel) and link the in-tree shared library."""
    if not force and not needs_build():
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    nvcc = _nvcc()
    with tempfile.TemporaryDirectory(prefix="b200_build_") as tmp_dir:
        units = sorted(CSRC.glob("*.cu"))
        objects = [Path(tmp_dir) / (u.stem + ".o") for u in units]
        cmds = [[nvcc, *NVCC_FLAGS, "-c", "-o", str(o), str(u)] for u, o in zip(units, objects)]
        tmp = LIB_PATH.with_suffix(".so.tmp")
        link = [nvcc, *NVCC_FLAGS[:2], "-shared", "-o", str(tmp), *map(str, objects)]
        with concurrent.futures.ThreadPoolExecutor(len(cmds)) as pool:
            procs = list(pool.map(lambda c: subprocess.run(c, capture_output=True, text=True), cmds))
        if all(p.returncode == 0 for p in procs):
            cmds.append(link)
            procs.append(subprocess.run(link, capture_output=True, text=True))
    log = "".join(" ".join(c) + "\n" + p.stdout + p.stderr for c, p in zip(cmds, procs))
    (LIB_DIR / "build.log").write_text(log)
    failed = [p.returncode for p in procs if p.returncode != 0]
    if failed:
        sys.stderr.write(log)
        raise RuntimeError(f"nvcc failed building {LIB_PATH.name} (exit {failed[0]})")
    if verbose:
        sys.stdout.write(log)
    tmp.replace(LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))

"""Builds ``libmoe_b200.so`` (sm_100a) from the CUDA sources in this folder, and
the CPython binding of the layer-training entry points (``layer_binding.cpp``,
against the installed torch's headers).

Output: ``<package>/lib/libmoe_b200.so``.  nvcc cross-compiles for sm_100a
without a GPU.  The build is skipped when the library is newer than every
source and header.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
REPO = PKG.parent
LIB_DIR = PKG / "lib"
LIB = LIB_DIR / "libmoe_b200.so"
OBJ_DIR = PKG / "_build"
SOURCES = ["moe_b200.cu", "layer_train.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _deps() -> list[Path]:
    files = [p for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh", ".h")]
    files += list((REPO / "include").glob("*.h"))
    return files


def build(force: bool = False, verbose: bool = False) -> Path:
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    if LIB.exists() and not force:
        lib_t = LIB.stat().st_mtime
        if all(p.stat().st_mtime <= lib_t for p in _deps()):
            return LIB
    tmp = LIB.with_suffix(".so.tmp")
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    flags = [*ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-O2", "-I", str(REPO / "include")]
    if verbose:
        flags.insert(0, "-Xptxas=-v")
    newest_header = max(p.stat().st_mtime for p in _deps() if p.suffix != ".cu")
    jobs, objects = [], []
    for name in SOURCES:  # one nvcc per source, side by side; objects newer than their inputs are kept
        src, obj = CSRC / name, OBJ_DIR / (name + ".o")
        objects.append(str(obj))
        if not force and obj.exists() and obj.stat().st_mtime > max(newest_header, src.stat().st_mtime):
            continue
        cmd = [_nvcc(), *flags, "-c", "-o", str(obj), str(src)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        jobs.append((cmd, subprocess.Popen(cmd, cwd=str(CSRC))))
    for cmd, job in jobs:
        if job.wait():
            raise subprocess.CalledProcessError(job.returncode, cmd)
    subprocess.run([_nvcc(), *ARCH, "-shared", "-o", str(tmp), *objects], check=True, cwd=str(CSRC))
    os.replace(tmp, LIB)
    return LIB


def native_path() -> Path:
    import torch
    return LIB_DIR / f"moe_layer_native.{sys.implementation.cache_tag}-torch{torch.__version__}.so"


def build_native(force: bool = False) -> Path:
    """The binding ``src/_lib.py::native`` loads; one per Python and torch version."""
    import torch
    out, src = native_path(), CSRC / "layer_binding.cpp"
    inputs = [src, REPO / "include" / "moe_b200.h"]
    if out.exists() and not force and all(p.stat().st_mtime <= out.stat().st_mtime for p in inputs):
        return out
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    dirs = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
            REPO / "include"]
    tmp = out.with_suffix(".so.tmp")
    cmd = [shutil.which("g++") or "g++", "-O2", "-fPIC", "-shared", "-std=c++17",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", sysconfig.get_paths()["include"]]
    for d in dirs:
        cmd += ["-isystem", str(d)]
    cmd += [str(src), "-o", str(tmp), "-L", str(root / "lib")]
    # The shared C++ library by name: a compiler set up to link it statically
    # would give the module streams of its own, apart from those torch set up.
    cmd += ["-l:libstdc++.so.6"]
    cmd += [f"-l{name}" for name in ("torch_python", "torch_cuda", "torch_cpu", "torch", "c10_cuda", "c10")]
    subprocess.run(cmd, check=True, cwd=str(CSRC))
    os.replace(tmp, out)
    return out


if __name__ == "__main__":
    out = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(out)
    print(build_native(force="--force" in sys.argv))

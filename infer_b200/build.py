"""Build recipe of libinfer_b200.so (sm_100a only) and of the host module _host_ops.so.

``python -m infer_b200.build`` compiles every ``csrc/*.cu`` with nvcc into one shared
library next to this file, and ``csrc/host_ops.cpp`` with g++ against PyTorch's headers into
a Python module beside it.  Either is rebuilt only when a source is newer than it.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "libinfer_b200.so"
HOST_OPS = HERE / "_host_ops.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def sources():
    return sorted(CSRC.glob("*.cu"))


def _stale() -> bool:
    if not LIB.exists():
        return True
    newest = max(p.stat().st_mtime for p in list(CSRC.glob("*")) + [HERE.parent / "include" / "infer_b200.h"])
    return newest > LIB.stat().st_mtime


def build_host_ops(force: bool = False) -> subprocess.Popen | None:
    """Starts the compiler on host_ops.cpp; None when the module is up to date."""
    src = CSRC / "host_ops.cpp"
    newest = max(p.stat().st_mtime for p in [src, *(HERE.parent / "include").glob("infer_b200*.h")])
    if not force and HOST_OPS.exists() and HOST_OPS.stat().st_mtime >= newest:
        return None
    import sysconfig
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in (root / "include", root / "include/torch/csrc/api/include", sysconfig.get_paths()["include"],
                                f"{cuda}/include")),
           str(src), "-o", str(HOST_OPS), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def build(force: bool = False, verbose: bool = False) -> Path:
    host = build_host_ops(force)
    try:
        build_library(force, verbose)
    finally:
        if host is not None:
            out, _ = host.communicate()
            if host.returncode != 0 or verbose:
                sys.stderr.write(f"--- host_ops.cpp\n{out}\n")
    if host is not None and host.returncode != 0:
        raise RuntimeError("g++ failed")
    return LIB


def build_library(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    objs = []
    build_dir = HERE / "build"
    build_dir.mkdir(exist_ok=True)
    procs = []
    for src in sources():
        obj = build_dir / (src.stem + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(str(obj))
    failed = False
    for src, proc in procs:
        out, _ = proc.communicate()
        if proc.returncode != 0 or verbose:
            sys.stderr.write(f"--- {src.name}\n{out}\n")
        failed |= proc.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    subprocess.check_call([nvcc, "-shared", "-o", str(LIB), *objs, "-gencode", "arch=compute_100a,code=sm_100a"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))

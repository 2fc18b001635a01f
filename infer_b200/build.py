"""Build recipe of libinfer_b200.so (sm_100a only) and of the host module _host_ops.so.

``python -m infer_b200.build`` compiles every ``csrc/*.cu`` with nvcc into one shared
library next to this file, and ``csrc/host_ops.cpp`` with g++ against PyTorch's headers into
a Python module beside it.  Either is rebuilt only when a source of its own is newer than it, the
module also when it was built for another PyTorch or Python.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "libinfer_b200.so"
HOST_OPS = HERE / "_host_ops.so"
HOST_OPS_TARGET = HERE / "_host_ops.target"      # what the module was built for

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
    own = [*sources(), *CSRC.glob("*.cuh"), *(HERE.parent / "include").glob("infer_b200*.h"), HERE.parent / "include" / "block_manager.hpp"]
    return max(p.stat().st_mtime for p in own) > LIB.stat().st_mtime


def host_ops_target() -> str:
    """The PyTorch and the Python that a module built now fits."""
    import torch
    return f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"


def _host_ops_stale(target: str) -> bool:
    if not HOST_OPS.exists() or not HOST_OPS_TARGET.exists() or HOST_OPS_TARGET.read_text() != target:
        return True
    own = [CSRC / "host_ops.cpp", *(HERE.parent / "include").glob("infer_b200*.h")]
    return max(p.stat().st_mtime for p in own) > HOST_OPS.stat().st_mtime


def build_host_ops(force: bool = False) -> subprocess.Popen | None:
    """Starts the compiler on host_ops.cpp; None when the module is up to date."""
    src, target = CSRC / "host_ops.cpp", host_ops_target()
    if not force and not _host_ops_stale(target):
        return None
    HOST_OPS_TARGET.unlink(missing_ok=True)
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
    host, why = None, ""
    try:
        host = build_host_ops(force)
    except (ImportError, OSError) as e:          # no PyTorch or no compiler: the library is built all the same
        why = str(e)
    try:
        build_library(force, verbose)
    finally:
        if host is not None:
            out, _ = host.communicate()
            if host.returncode != 0 or verbose:
                sys.stderr.write(f"--- host_ops.cpp\n{out}\n")
            if host.returncode == 0:
                HOST_OPS_TARGET.write_text(host_ops_target())
            else:
                why = "g++ failed"
    if why:
        raise RuntimeError(f"{LIB.name} is built, {HOST_OPS.name} is not, and the ops that it launches will refuse: {why}")
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

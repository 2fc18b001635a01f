"""When the build recipe compiles what, on empty files in a folder of its own."""
import os

import pytest

from infer_b200 import build


class Compiler:
    """Stands in for subprocess.Popen: writes the output file, or fails."""
    ran, fails = [], ()

    def __init__(self, cmd, **kw):
        Compiler.ran.append(os.path.basename(cmd[cmd.index("-o") + 1]))
        self.returncode = 1 if Compiler.ran[-1] in Compiler.fails else 0
        if self.returncode == 0:
            open(cmd[cmd.index("-o") + 1], "w").close()

    def communicate(self):
        return "", None


@pytest.fixture
def tree(tmp_path, monkeypatch):
    here = tmp_path / "infer_b200"
    files = [here / "csrc" / "a.cu", here / "csrc" / "a.cuh", here / "csrc" / "host_ops.cpp", tmp_path / "include" / "infer_b200.h",
             tmp_path / "include" / "block_manager.hpp"]
    for f in files:
        f.parent.mkdir(parents=True, exist_ok=True)
        f.write_text("")
        os.utime(f, (1000, 1000))
    Compiler.ran, Compiler.fails = [], ()
    for name, value in (("HERE", here), ("CSRC", here / "csrc"), ("LIB", here / "libinfer_b200.so"), ("HOST_OPS", here / "_host_ops.so"),
                        ("HOST_OPS_TARGET", here / "_host_ops.target")):
        monkeypatch.setattr(build, name, value, raising=False)
    monkeypatch.setattr(build.subprocess, "Popen", Compiler)
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: Compiler(cmd))

    def again(touched=None):
        Compiler.ran = []
        for f in here.glob("*.so"):
            os.utime(f, (2000, 2000))
        if touched:
            os.utime(tmp_path / touched, (3000, 3000))
        build.build()
        return sorted(Compiler.ran)

    build.build()
    assert sorted(Compiler.ran) == ["_host_ops.so", "a.o", "libinfer_b200.so"]
    assert again() == []
    return again


def test_the_host_module_is_built_again_for_another_pytorch(tree, monkeypatch):
    import torch
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    assert tree() == ["_host_ops.so"]
    assert tree() == []


def test_either_is_rebuilt_for_its_own_sources_alone(tree):
    assert tree("infer_b200/csrc/host_ops.cpp") == ["_host_ops.so"]
    assert tree("infer_b200/csrc/host_ops.cpp") == ["_host_ops.so"]         # older than the file still
    os.utime(build.CSRC / "host_ops.cpp", (1000, 1000))
    assert tree("infer_b200/csrc/a.cuh") == ["a.o", "libinfer_b200.so"]
    os.utime(build.CSRC / "a.cuh", (1000, 1000))
    assert tree("include/infer_b200.h") == ["_host_ops.so", "a.o", "libinfer_b200.so"]


@pytest.mark.parametrize("how", ["compiler fails", "no compiler", "no pytorch"])
def test_the_library_is_built_where_the_host_module_cannot_be(tree, monkeypatch, how):
    build.LIB.unlink()
    build.HOST_OPS.unlink()
    Compiler.ran = []
    if how == "compiler fails":
        Compiler.fails = ("_host_ops.so",)
    else:
        def missing(force):
            raise FileNotFoundError("g++") if how == "no compiler" else ImportError("torch")
        monkeypatch.setattr(build, "build_host_ops", missing)
    with pytest.raises(RuntimeError, match="_host_ops.so"):
        build.build()
    assert build.LIB.exists() and not build.HOST_OPS.exists()
    if how == "compiler fails":                                             # a failed build is not taken for a finished one
        Compiler.fails = ()
        assert tree() == ["_host_ops.so"]

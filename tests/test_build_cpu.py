"""The build recipe's choices: what is stale, and what is built where torch is missing.  Nothing is compiled here."""

import os
import sys
from pathlib import Path

import pytest

from maxsim_b200 import build


class _Process:
    returncode = 0

    def __init__(self, cmd, **kw):
        _write(cmd)

    def communicate(self):
        return b"", None


def _write(cmd, **kw):
    Path(cmd[cmd.index("-o") + 1]).write_text("built")


@pytest.fixture
def package(tmp_path, monkeypatch):
    """A package folder of its own, compilers that only write their output, and the commands they were given."""
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in ("a.cu", "b.cu", "c.cuh", "generation_binding.cpp"):
        (csrc / name).write_text("")
    (tmp_path / "nvcc").write_text("")
    ran = []
    for name, value in (("PKG", tmp_path), ("CSRC", csrc), ("LIB", tmp_path / "libmaxsim_b200.so"),
                        ("BINDING_SRC", csrc / "generation_binding.cpp"), ("BINDING", tmp_path / "_generation.so")):
        monkeypatch.setattr(build, name, value)
    monkeypatch.setenv("NVCC", str(tmp_path / "nvcc"))
    monkeypatch.setattr(build.subprocess, "Popen", lambda cmd, **kw: ran.append(cmd) or _Process(cmd, **kw))
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or _write(cmd, **kw))
    return ran


def _later(path, seconds=10):
    now = max(p.stat().st_mtime for p in build.PKG.rglob("*") if p.is_file())
    os.utime(path, (now + seconds, now + seconds))


def test_the_library_builds_without_torch(package, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # what `import torch` finds where it is not installed
    assert build.needs_build()
    assert build.build() == build.LIB and build.LIB.exists() and not build.BINDING.exists()
    assert "torch" in capsys.readouterr().err
    assert not build.needs_build()
    del package[:]
    build.build()
    assert package == []
    _later(build.CSRC / "generation_binding.cpp")  # of no concern without torch
    assert not build.needs_build()


def test_torch_that_comes_later_brings_the_module(package, monkeypatch):
    pytest.importorskip("torch")
    with monkeypatch.context() as without:
        without.setitem(sys.modules, "torch", None)
        build.build()
    assert build.needs_build()
    del package[:]
    build.build()
    assert build.BINDING.exists() and not build.needs_build()
    assert len(package) == 1 and "generation_binding.cpp" in " ".join(package[0])  # the library was not built again


def test_another_torch_makes_the_module_stale(package, monkeypatch):
    pytest.importorskip("torch")
    build.build()
    assert not build.needs_build()
    monkeypatch.setattr(build, "torch_build", lambda: "another torch")
    assert build.needs_build()


def test_sources_make_stale_what_they_go_into(package):
    pytest.importorskip("torch")
    build.build()
    for name, commands in (("generation_binding.cpp", 1), ("c.cuh", 3), ("b.cu", 3)):
        _later(build.CSRC / name)
        assert build.needs_build()
        del package[:]
        build.build()
        assert len(package) == commands  # the module alone; or two sources and the library that the module loads
        for path in (build.LIB, build.BINDING):
            _later(path)
        assert not build.needs_build()

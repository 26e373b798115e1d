"""The native build on a machine that lacks something, with the compilers faked."""

from __future__ import annotations

import os

import pytest

from diffucore_b200 import build


@pytest.fixture
def compilers(monkeypatch, tmp_path):
    """Commands are recorded and leave an empty output file; everything built lies in tmp_path."""
    ran = []

    def run(cmd, verbose):
        ran.append(cmd[0].rsplit("/", 1)[-1])
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "_nvcc", lambda: "nvcc")
    for name in ("LIB", "EXT", "OBJECTS"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    return ran


def test_builds_both(compilers, monkeypatch):
    monkeypatch.setattr(build, "ext_missing", lambda: None)
    assert build.build() == build.LIB and build.LIB.exists() and build.EXT.exists()
    assert compilers == ["nvcc"] * 3 + ["g++"]
    build.build()
    assert len(compilers) == 4                              # up to date


@pytest.mark.parametrize("lacks", ["g++", "Python.h", "torch/extension.h"])
def test_library_alone_without_what_the_binding_needs(compilers, monkeypatch, capsys, tmp_path, lacks):
    which, includes = build.shutil.which, build._ext_includes()
    if lacks == "g++":
        monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else which(name))
    else:
        monkeypatch.setattr(build, "_ext_includes", lambda: [d for d in includes if not os.path.exists(d / lacks)])
    assert build.build() == build.LIB and build.LIB.exists() and not build.EXT.exists()
    assert compilers == ["nvcc"] * 3
    assert f"{lacks} not found" in capsys.readouterr().err


def test_binding_is_rebuilt_for_another_torch(compilers, monkeypatch):
    monkeypatch.setattr(build, "ext_missing", lambda: None)
    build.build()
    stamp = build._ext_stamp()
    monkeypatch.setattr(build, "_ext_stamp", lambda: stamp.replace("torch ", "torch 0."))
    build.build()
    assert compilers[4:] == ["g++"]
    build.build()
    assert len(compilers) == 5

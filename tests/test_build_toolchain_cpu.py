"""The build where parts of the toolchain are absent, and what makes the binding out of date (commands are recorded, not run)."""
from __future__ import annotations

import importlib.util
import os
import shutil
import sys

import pytest

from cuda_gpt2_inference_b200 import build


@pytest.fixture()
def recorded(monkeypatch, tmp_path):
    """build.build() into empty folders; every command 'succeeds' by making its output."""
    ran = []

    def run(cmd, verbose=False):
        ran.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("")
        return ""

    monkeypatch.setattr(build, "_run", run)
    for name, path in (("OBJ", "_build"), ("LIB", "libgpt2b.so"), ("BIND", "_bind.so"), ("BIND_FOR", "_build/bind_for.txt")):
        monkeypatch.setattr(build, name, str(tmp_path / path), raising=False)
    return ran


def _made(ran, path):
    return [c for c in ran if c[c.index("-o") + 1] == path]


def test_library_is_linked_without_torch(recorded, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build() == build.LIB
    assert len(_made(recorded, build.LIB)) == 1 and not _made(recorded, build.BIND)
    assert "_bind.so left out: no torch here" in capsys.readouterr().err


@pytest.mark.parametrize("what", ["g++", "Python's headers"])
def test_library_is_linked_without_what_only_the_binding_needs(recorded, monkeypatch, tmp_path, capsys, what):
    if what == "g++":
        monkeypatch.setattr(shutil, "which", lambda name, *a, **k: None)
    else:
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "none")})
    assert build.build() == build.LIB
    assert len(_made(recorded, build.LIB)) == 1 and not _made(recorded, build.BIND)
    assert f"no {what} here" in capsys.readouterr().err


def test_library_is_linked_though_the_binding_fails(recorded, monkeypatch):
    run = build._run

    def failing(cmd, verbose=False):
        if cmd[cmd.index("-o") + 1] == build.BIND:
            raise RuntimeError("g++ failed")
        return run(cmd, verbose)

    monkeypatch.setattr(build, "_run", failing)
    with pytest.raises(RuntimeError, match="g"):
        build.build()
    assert os.path.exists(build.LIB)


def test_binding_follows_torch_and_python(recorded, monkeypatch):
    build.build()
    assert len(_made(recorded, build.BIND)) == 1
    build.build()
    assert len(_made(recorded, build.BIND)) == 1  # nothing changed
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "99.0")
    build.build()
    assert len(_made(recorded, build.BIND)) == 2
    monkeypatch.setattr(sys, "version", "4.0")
    build.build()
    build.build()
    assert len(_made(recorded, build.BIND)) == 3


def test_a_failed_command_is_named(tmp_path):
    with pytest.raises(RuntimeError, match="^g\\+\\+ failed"):
        build._run(["g++", str(tmp_path / "none.cpp"), "-o", str(tmp_path / "x")])

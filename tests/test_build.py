"""CPU tests of the build's order and of what it needs: no compiler is run."""

import os
import subprocess

import pytest

from mxfp4_b200 import build


@pytest.fixture
def ran(monkeypatch, tmp_path):
    """Outputs in an empty folder; the compilers' commands are recorded, and each writes its output."""
    monkeypatch.setattr(build, "OUT", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "BINDING_OUT", str(tmp_path / "_attention.so"))
    commands, codes = [], {}

    def run(cmd, **_):
        what = "binding" if build.BINDING in cmd else "library"
        commands.append(what)
        if codes.get(what, 0) == 0:
            with open(cmd[cmd.index("-o") + 1], "wb") as f:
                f.write(" ".join(cmd).encode().replace(b'"', b"\0"))
        return subprocess.CompletedProcess(cmd, codes.get(what, 0), "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    return commands, codes


def test_the_library_is_built_first(ran):
    commands, _ = ran
    assert build.build() == build.OUT and commands == ["library", "binding"]
    assert os.path.exists(build.OUT) and os.path.exists(build.BINDING_OUT)


def test_a_host_without_what_the_binding_needs_builds_the_library(ran, monkeypatch, capsys):
    commands, _ = ran
    monkeypatch.setattr(build, "binding_needs", lambda: ["torch", "Python.h"])
    assert build.build() == build.OUT and commands == ["library"]
    assert "torch, Python.h" in capsys.readouterr().err


def test_needs_are_found(monkeypatch, tmp_path):
    assert build.binding_needs() == []
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    assert build.binding_needs() == ["a host C++ compiler"]
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.binding_needs() == ["Python.h", "a host C++ compiler"]


def test_a_failing_host_compiler_is_an_error_after_the_library(ran):
    commands, codes = ran
    codes["binding"] = 1
    with pytest.raises(RuntimeError, match="_attention.so"):
        build.build()
    assert os.path.exists(build.OUT) and commands == ["library", "binding"]


def test_a_binding_for_another_torch_or_python_is_built_again(ran, monkeypatch):
    commands, _ = ran
    build.build()
    build.build()
    assert commands == ["library", "binding"]
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399-x86_64-linux-gnu")
    build.build()
    assert commands == ["library", "binding", "binding"]
    import torch

    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    build.build()
    assert commands == ["library", "binding", "binding", "binding"]


def test_a_binding_for_another_torch_is_refused(monkeypatch):
    """Before it is loaded: its view of a tensor is another one."""
    import torch

    from mxfp4_b200 import attention

    assert build.binding_fits()
    monkeypatch.setattr(attention, "_native", None)
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    with pytest.raises(RuntimeError, match="another torch or Python"):
        attention._binding()
    assert attention._native is None

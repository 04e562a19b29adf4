"""The build on hosts that lack something, and after a change of torch (no compiler runs here)."""

from __future__ import annotations

import importlib.metadata
import importlib.util
import subprocess
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "llm-serving_b200" / "build.py"


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py over an empty output folder, its commands recorded and their outputs touched instead of run."""
    spec = importlib.util.spec_from_file_location("build_under_test", SOURCE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "BUILD", tmp_path)
    monkeypatch.setattr(module, "LIB", tmp_path / "libpaged_decode.so")
    monkeypatch.setattr(module, "OPS", tmp_path / "pd_ops.so")
    monkeypatch.setattr(module, "OPS_STAMP", tmp_path / "pd_ops.stamp", raising=False)
    module.commands, module.fails = [], set()

    def run(cmd, **_):
        out = Path(cmd[cmd.index("-o") + 1])
        module.commands.append(out.name)
        if out.name in module.fails:
            return subprocess.CompletedProcess(cmd, 1, "", "error")
        out.touch()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(module.subprocess, "run", run)
    return module


def test_everything_once_and_then_nothing(build):
    assert build.build() == build.LIB and build.LIB.exists() and build.OPS.exists()
    assert len(build.commands) == len(build.SOURCES) + 2
    build.commands.clear()
    build.build()
    assert build.commands == []


def test_without_torch_the_library_is_built_alone(build, monkeypatch, capsys):
    build.OPS.touch()  # another torch's
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build().exists() and not build.OPS.exists()
    assert "torch is not installed" in capsys.readouterr().err


def test_without_a_host_compiler_the_library_is_built_alone(build, monkeypatch, capsys):
    monkeypatch.setattr("shutil.which", lambda name, *a, **k: None)
    assert build.build().exists() and "pd_ops.so" not in build.commands
    assert "g++" in capsys.readouterr().err


def test_a_binding_that_does_not_compile_is_an_error_but_the_library_stands(build):
    build.fails.add("pd_ops.so")
    with pytest.raises(RuntimeError, match="failed"):
        build.build()
    assert build.LIB.exists()
    build.fails.clear()
    build.commands.clear()
    build.build()
    assert build.commands == ["pd_ops.so"]


def test_another_torch_rebuilds_the_binding(build, monkeypatch):
    build.build()
    build.commands.clear()
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0" if name == "torch" else version(name))
    build.build()
    assert build.commands == ["pd_ops.so"]

"""The build of the native parts, with compilers that only leave a mark."""
import subprocess
import time

import pytest

from sandmuon_b200.csrc import build


@pytest.fixture
def compilers(tmp_path, monkeypatch):
    """nvcc as a script that notes its start and runs for a minute, and targets
    of their own."""
    started = tmp_path / "started"
    nvcc = tmp_path / "bin" / "nvcc"
    nvcc.parent.mkdir()
    nvcc.write_text(f"#!/bin/sh\necho $$ >> {started}\nexec sleep 60\n")
    nvcc.chmod(0o755)
    monkeypatch.setattr(build, "nvcc_path", lambda: str(nvcc))
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / "lib.so")
    return started


def alive(started):
    pids = [int(line) for line in started.read_text().split()] if started.exists() else []
    return [pid for pid in pids if subprocess.run(["kill", "-0", str(pid)], capture_output=True).returncode == 0]


def test_no_compiler_starts_when_another_is_missing(compilers, monkeypatch):
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    with pytest.raises(RuntimeError, match="g\\+\\+ not found"):
        build.build(force=True)
    time.sleep(0.5)
    assert not alive(compilers)


def test_no_compiler_is_left_behind_when_another_does_not_start(compilers, tmp_path, monkeypatch):
    monkeypatch.setattr(build, "binding_command", lambda out: [str(tmp_path / "nothing")])
    with pytest.raises(FileNotFoundError):
        build.build(force=True)
    time.sleep(0.5)
    assert not alive(compilers)


def test_the_extension_of_another_torch_is_not_taken(built_library, monkeypatch):
    """The extension is kept and loaded for the torch it was built with alone."""
    from sandmuon_b200 import _lib
    asked = []
    monkeypatch.setattr(build, "binding_command", lambda out: asked.append(out) or ["true"])
    build.build()
    assert not asked and _lib.binding() is not None
    monkeypatch.setattr(build.os, "replace", lambda *_: None)
    monkeypatch.setattr("torch.__version__", "0.0.0+other")
    build.build()
    assert len(asked) == 1 and "0.0.0+other" in asked[0].name
    monkeypatch.setattr(_lib, "_binding", None)
    with pytest.raises(RuntimeError, match="not built"):
        _lib.binding()

"""The torch calls are rebuilt when their source or the torch they are for
changes (g++ replaced by a stand-in)."""

import os
import subprocess

import pytest
import torch

from quail_b200 import build


@pytest.fixture
def compiles(monkeypatch, tmp_path):
    """The number of compilations so far; the build goes to a folder of its own."""
    monkeypatch.setattr(build, "TORCH_OPS", tmp_path / "_torch_ops.so")
    monkeypatch.setattr(build, "BUILD_DIR", tmp_path / "build")
    (tmp_path / "build").mkdir()
    done = []

    def run(cmd, **_):
        done.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(build.subprocess, "run", run)
    return done


def test_built_once(compiles):
    for _ in range(3):
        build._build_torch_ops(False)
    assert len(compiles) == 1
    build._build_torch_ops(True)
    assert len(compiles) == 2


@pytest.mark.parametrize("change", ["torch", "python"])
def test_another_torch_or_python_is_stale(compiles, monkeypatch, change):
    build._build_torch_ops(False)
    if change == "torch":
        monkeypatch.setattr(torch, "__version__", "2.99.0")
    else:
        monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399-x86_64")
    build._build_torch_ops(False)
    build._build_torch_ops(False)
    assert len(compiles) == 2


def test_a_build_of_unknown_origin_is_stale(compiles):
    """A library from before its torch was recorded."""
    build.TORCH_OPS.write_text("built")
    os.utime(build.TORCH_OPS, (2 ** 31, 2 ** 31))
    build._build_torch_ops(False)
    assert len(compiles) == 1

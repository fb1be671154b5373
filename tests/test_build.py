"""What the build makes of an environment: the C library needs neither torch nor a host compiler, and the Python module follows torch."""
import os
import subprocess
import sys
import sysconfig

import pytest

from thunderkittens_b200 import build


@pytest.fixture
def compiles(monkeypatch, tmp_path):
    """The commands that the build of the module would run, in a folder of its own; a command leaves its output file."""
    torch_ops = getattr(build, "TORCH_OPS")
    monkeypatch.setattr(build, "TORCH_OPS", str(tmp_path / os.path.basename(torch_ops)))
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    seen = []

    def run(cmd, **kwargs):
        seen.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    return seen


def test_without_torch(compiles, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    build._build_torch_ops(False)
    assert compiles == [] and "no torch" in capsys.readouterr().err


def test_without_a_host_compiler(compiles, monkeypatch, tmp_path, capsys):
    monkeypatch.setenv("PATH", str(tmp_path))
    build._build_torch_ops(False)
    assert compiles == [] and "is not: no g++" in capsys.readouterr().err


def test_the_module_is_built_again_for_another_torch(compiles, monkeypatch):
    import torch
    build._build_torch_ops(False)
    build._build_torch_ops(False)
    assert len(compiles) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build._build_torch_ops(False)
    assert len(compiles) == 2 and any("9.9.9" in a for a in compiles[1])
    build._build_torch_ops(False)
    assert len(compiles) == 2


def test_the_module_is_named_after_its_python():
    assert build.TORCH_OPS.endswith(sysconfig.get_config_var("EXT_SUFFIX"))


def test_a_module_of_another_torch_is_refused(lib, monkeypatch):
    import torch
    from thunderkittens_b200 import ops
    assert ops._native().torch_version == torch.__version__
    monkeypatch.setattr(ops, "_torch_ops", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(ImportError, match="9.9.9"):
        ops._native()

"""build.py without what only the Python package's host extension needs: the library is linked all the same."""
import importlib.util
import os
import subprocess
import sys

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "startlux-prism_amd", "build.py")


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The module with its outputs under tmp_path, hipcc replaced by one that leaves an empty file, and an older extension
    in place; programs other than hipcc run as they are."""
    spec = importlib.util.spec_from_file_location("prism_build", PATH)
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    for name, at in (("OBJ", "obj"), ("LIB", "lib.so"), ("HOST", "host.so")):
        monkeypatch.setattr(b, name, str(tmp_path / at))
    open(b.HOST, "w").close()
    real = subprocess.run

    def run(cmd, **kw):
        if cmd[0] != b.HIPCC:
            return real(cmd, **kw)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(b.subprocess, "run", run)
    return b


def test_without_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch.utils", None)
    assert os.path.exists(build.build())
    assert not os.path.exists(build.HOST) and "is not built" in capsys.readouterr().err


def test_without_a_compiler(build, monkeypatch, tmp_path, capsys):
    monkeypatch.setenv("CXX", str(tmp_path / "none"))
    assert os.path.exists(build.build())
    assert not os.path.exists(build.HOST) and "is not built" in capsys.readouterr().err


def test_a_compiler_that_fails_is_an_error(build, monkeypatch):
    """... after the library is linked."""
    monkeypatch.setenv("CXX", "false")
    with pytest.raises(RuntimeError):
        build.build()
    assert os.path.exists(build.LIB)

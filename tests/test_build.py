"""What build() makes and when, with a compiler that only writes its output file."""
import os
import subprocess
import sys
import types

import pytest

from ferret_b200 import build as B


@pytest.fixture
def made(tmp_path, monkeypatch):
    """The build in tmp_path; a list of what was compiled or linked."""
    for name in ("LIB", "BIN", "HOST", "HOST_FOR", "BUILD"):
        if hasattr(B, name):
            monkeypatch.setattr(B, name, str(tmp_path / os.path.basename(getattr(B, name))))
    calls = []

    def run(cmd, **kw):
        target = cmd[cmd.index("-o") + 1]
        with open(target, "w") as f:
            f.write("x")
        calls.append(os.path.basename(target))
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return calls


def test_the_library_needs_no_torch(made, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)       # import torch fails
    assert B.build() == B.LIB and os.path.exists(B.LIB) and os.path.exists(B.BIN)
    assert not os.path.exists(B.HOST) and "torch" in capsys.readouterr().err
    del made[:]
    assert B.build() == B.LIB and made == []              # and that is all there is to do
    assert B.build(force=True) == B.LIB and not os.path.exists(B.HOST)


@pytest.mark.parametrize("absent", ["g++", "Python.h"])
def test_the_library_needs_no_host_toolchain(made, monkeypatch, capsys, absent):
    if absent == "g++":
        real = B.shutil.which
        monkeypatch.setattr(B.shutil, "which", lambda p: None if p == "g++" else real(p))
    else:
        paths = dict(B.sysconfig.get_paths(), include="/nonexistent")
        monkeypatch.setattr(B.sysconfig, "get_paths", lambda: paths)
    assert B.build() == B.LIB and os.path.exists(B.LIB) and not os.path.exists(B.HOST)
    assert "not built" in capsys.readouterr().err


def test_the_module_follows_the_installed_torch(made, monkeypatch):
    B.build()
    assert os.path.exists(B.LIB) and os.path.exists(B.HOST)
    del made[:]
    B.build()
    assert made == []
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "0.0.other")
    B.build()
    assert made == [os.path.basename(B.HOST) + ".tmp"]    # the module alone
    del made[:]
    B.build()
    assert made == []


def test_the_module_is_made_alone_when_it_is_missing(made):
    B.build()
    os.remove(B.HOST)
    del made[:]
    B.build()
    assert made == [os.path.basename(B.HOST) + ".tmp"]

"""The library for hosts without torch is built whatever becomes of the Python
side's checking module (compilers faked: nothing is compiled here)."""
import os
import subprocess
import sys

import pytest

from tinygpt_amd import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    for name, file in (("OUT", "lib.so"), ("FLOOR_OUT", "floor.so"), ("PY_OUT", "calls.so")):
        monkeypatch.setattr(b, name, str(tmp_path / file))
    monkeypatch.setattr(b, "HERE", str(tmp_path))
    return tmp_path


def compilers(monkeypatch, calls):
    """Every command writes its output file; the checking module's does what `calls` does."""
    def run(cmd, **kw):
        if any(str(x).endswith(b.PY_SRC) for x in cmd):
            return calls(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b.subprocess, "run", run)


def missing(cmd):
    raise FileNotFoundError(cmd[0])


def failing(cmd):
    return subprocess.CompletedProcess(cmd, 1, "", "no such header")


def test_without_torch(tree, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    monkeypatch.setitem(sys.modules, "torch.utils", None)
    compilers(monkeypatch, failing)
    assert b.build() == b.OUT
    assert os.path.exists(b.OUT) and os.path.exists(b.FLOOR_OUT) and not os.path.exists(b.PY_OUT)


@pytest.mark.parametrize("calls", [missing, failing])
def test_without_a_compiler_for_the_checks(tree, monkeypatch, calls):
    compilers(monkeypatch, calls)
    with pytest.raises(RuntimeError, match=b.PY_SRC):
        b.build()
    assert os.path.exists(b.OUT) and os.path.exists(b.FLOOR_OUT) and not os.path.exists(b.PY_OUT)

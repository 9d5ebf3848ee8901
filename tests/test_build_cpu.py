"""The build's order, with the compilers replaced: the C library and the native
harness do not depend on the extension module."""
import subprocess
import sys
from pathlib import Path

import pytest

from neso_b200 import build


@pytest.fixture
def tools(tmp_path, monkeypatch):
    """Paths under tmp_path, compilers that write an empty output; returns the commands' outputs."""
    made = []

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        made.append(out.name)
        if out.name == "_bindings.so.tmp":
            return subprocess.CompletedProcess(cmd, 1, "", "Python.h: No such file")
        out.write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    for name, file in (("BUILD", "_build"), ("LIB", "libneso_b200.so"), ("HARNESS", "neso_harness"), ("BINDING", "_bindings.so")):
        monkeypatch.setattr(build, name, tmp_path / file)
    return made


def test_library_and_harness_are_built_where_the_module_fails(tools):
    with pytest.raises(RuntimeError, match="Python.h"):
        build.build()
    assert build.LIB.exists() and build.HARNESS.exists() and not build.BINDING.exists()
    assert {"fa2.o", "libneso_b200.so.tmp", "neso_harness", "_bindings.so.tmp"} <= set(tools)


def test_library_and_harness_are_built_without_torch(tools, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB
    assert build.LIB.exists() and build.HARNESS.exists() and "_bindings.so.tmp" not in tools
    assert "_bindings.so is not built" in capsys.readouterr().err

"""What the build asks for, with the compilers replaced by stand-ins that leave empty files."""
import importlib.util
import subprocess
import sysconfig
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "edge-infer_b200"


@pytest.fixture
def builder(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("builder_under_test", PACKAGE / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.commands = []

    def run(command, **_):
        module.commands.append(command)
        Path(command[command.index("-o") + 1]).write_bytes(b"")
        return subprocess.CompletedProcess(command, 0, "", "")

    monkeypatch.setattr(module.subprocess, "run", run)
    package = tmp_path / "package"
    package.mkdir()
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "edge_infer_b200.h").write_text("")
    for name in ("HERE", "OBJ", "LIB", "CALLS"):
        monkeypatch.setattr(module, name, package / Path(getattr(module, name)).relative_to(PACKAGE))
    return module


def test_the_library_needs_no_python_headers(builder, tmp_path, monkeypatch, capsys):
    """A host that only links the library builds without them; the second build finds everything in place."""
    paths = dict(sysconfig.get_paths(), include=str(tmp_path / "nowhere"))
    monkeypatch.setattr(builder.sysconfig, "get_paths", lambda: paths)
    assert builder.build() == builder.LIB and builder.LIB.exists()
    assert not any("python_calls" in part for command in builder.commands for part in command)
    assert "Python.h" in capsys.readouterr().err
    builder.commands.clear()
    builder.build()
    assert builder.commands == []


def test_python_calls_are_built_for_one_interpreter(builder):
    """Their file's name carries the interpreter's suffix, and a build leaves none that any interpreter would load."""
    (builder.HERE / "_calls.so").write_bytes(b"")
    builder.build()
    assert (builder.HERE / ("_calls" + sysconfig.get_config_var("EXT_SUFFIX"))).exists()
    assert sysconfig.get_config_var("EXT_SUFFIX") == ".so" or not (builder.HERE / "_calls.so").exists()
    builder.commands.clear()
    builder.build()
    assert builder.commands == []

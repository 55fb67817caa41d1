"""The CPython binding belongs to one interpreter, and a C user needs none of it."""
import importlib.machinery as machinery
import subprocess
import sysconfig

import pytest

from cormorant_b200 import build, kernels


def test_binding_is_named_for_its_interpreter():
    build.build_binding()
    assert build.BIND.name == "_bind" + sysconfig.get_config_var("EXT_SUFFIX") and build.BIND.exists()
    assert kernels._native().__file__ == str(build.BIND)


@pytest.mark.parametrize("suffixes", [[".cpython-399-x86_64-linux-gnu.so", ".abi3.so", ".so"]])
def test_another_interpreter_finds_none(suffixes):
    build.build_binding()
    finder = machinery.FileFinder(str(build.PKG), (machinery.ExtensionFileLoader, suffixes))
    assert finder.find_spec("_bind") is None


def test_an_untagged_binding_is_taken_away(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "BIND", tmp_path / "_bind.tag.so")
    (tmp_path / "_bind.so").write_bytes(b"of an older build")
    assert build.build_binding() == build.BIND
    assert sorted(p.name for p in tmp_path.iterdir()) == ["_bind.tag.so"]


@pytest.mark.parametrize("missing", ["Python.h", "compiler"])
def test_without_the_means_there_is_no_binding_but_a_library(tmp_path, monkeypatch, capsys, missing):
    monkeypatch.setattr(build, "BIND", tmp_path / "_bind.tag.so")
    if missing == "Python.h":
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "none")})
    else:
        monkeypatch.setenv("CC", str(tmp_path / "no-such-compiler"))
    assert build.build_binding() is None and not build.BIND.exists()
    assert "_bind" in capsys.readouterr().err
    monkeypatch.setattr(build, "_stale", lambda target, deps: False)          # nothing else to compile
    assert build.build() == build.LIB


def test_a_failing_compiler_is_an_error(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "BIND", tmp_path / "_bind.tag.so")
    monkeypatch.setenv("CC", "false")
    with pytest.raises(subprocess.CalledProcessError):
        build.build_binding()

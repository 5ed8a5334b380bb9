"""What the build makes, and without what it can do (one small source in place of
the library's)."""

import ctypes
import shutil

import pytest

from einjax_amd.csrc import build


@pytest.fixture
def small(tmp_path, monkeypatch):
    try:
        build._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    (tmp_path / "one.hip").write_text('extern "C" int one() { return 1; }\n')
    monkeypatch.setattr(build, "BUILD_DIR", tmp_path / "_build")
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / "libejhip.so")
    monkeypatch.setattr(build, "TORCH_PATH", tmp_path / "_experts.so")
    monkeypatch.setattr(build, "sources", lambda: [tmp_path / "one.hip"])
    return tmp_path


def test_library_without_a_host_compiler(small, monkeypatch, capsys):
    (small / "_experts.so").write_text("of an earlier build")
    monkeypatch.setenv("HIPCC", build._hipcc())
    monkeypatch.setenv("PATH", str(small / "nothing"))
    assert build.build() == small / "libejhip.so"
    assert ctypes.CDLL(str(small / "libejhip.so")).one() == 1
    assert not (small / "_experts.so").exists()
    out, err = capsys.readouterr()
    assert "_experts.so" in err and "g++" in err and "_experts.so" not in out


def test_library_where_the_binding_fails(small, monkeypatch):
    """A binding that does not compile is an error, with the library in place."""
    if build.torch_binding_lacks():
        pytest.skip("the binding cannot be built here")
    (small / "bad.cpp").write_text("no C++\n")
    monkeypatch.setattr(build, "TORCH_SOURCE", small / "bad.cpp")
    with pytest.raises(RuntimeError, match="bad.cpp"):
        build.build()
    assert ctypes.CDLL(str(small / "libejhip.so")).one() == 1


def test_what_the_binding_lacks(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "_torch_root", lambda: None)
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    assert build.torch_binding_lacks() == ["g++", "Python's headers", "torch and its headers"]
    monkeypatch.undo()
    assert ("g++" in build.torch_binding_lacks()) == (shutil.which("g++") is None)

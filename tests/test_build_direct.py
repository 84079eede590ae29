"""CPU tests of the library's build where the Python module beside it cannot be built: the library is there all the same."""
import subprocess
import sys
import types

import pytest


@pytest.fixture
def lib(tmp_path, monkeypatch):
    """build_lib with its outputs in tmp_path, a hipcc that writes what it is told to, and a module of an earlier build."""
    import build_lib
    for name, at in (("BUILD", "_build"), ("LIB", "lib.so"), ("DIRECT", "direct.so")):
        monkeypatch.setattr(build_lib, name, tmp_path / at)
    build_lib.DIRECT.write_bytes(b"of another library")

    def run(cmd, **kw):
        if cmd[0] == hipcc:
            with open(cmd[cmd.index("-o") + 1], "wb") as f:
                f.write(b"library")
            return types.SimpleNamespace(returncode=0, stdout="", stderr="")
        return real(cmd, **kw)

    real, hipcc = subprocess.run, build_lib.HIPCC
    monkeypatch.setattr(subprocess, "run", run)
    return build_lib


def _check(lib, word):
    with pytest.warns(RuntimeWarning, match=word):
        assert lib.build() == lib.LIB
    assert lib.LIB.read_bytes() == b"library" and not lib.DIRECT.exists()


def test_without_a_compiler(lib, monkeypatch):
    monkeypatch.setattr(lib, "CXX", "no-such-compiler")
    _check(lib, "no-such-compiler")


def test_without_torch(lib, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    _check(lib, "torch")


def test_without_headers(lib, monkeypatch):
    monkeypatch.setattr(lib, "CXX", "false")  # a compiler that fails
    _check(lib, "direct.cpp")


def test_failed_library_leaves_both(lib, monkeypatch):
    lib.LIB.write_bytes(b"earlier")
    monkeypatch.setattr(lib, "HIPCC", "false")
    monkeypatch.setattr(lib, "CXX", "false")
    with pytest.raises(RuntimeError, match="hipcc failed|link failed"):
        lib.build()
    assert lib.LIB.read_bytes() == b"earlier" and lib.DIRECT.read_bytes() == b"of another library"

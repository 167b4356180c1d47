"""A binding that is missing, stale or does not compile costs host time, not the backend: the library is built and loaded
without it, and the calls that it serves go through the general path (no GPU needed)."""
import ctypes
import os
import subprocess
import sys
import types

import pytest
import torch

import versenext_amd
from versenext_amd import _lib, build


@pytest.fixture
def no_bind(monkeypatch):
    monkeypatch.setattr(_lib, "_bind", None)
    monkeypatch.delattr(versenext_amd, "_vnx_bind", raising=False)

    def put(module):
        monkeypatch.setitem(sys.modules, "versenext_amd._vnx_bind", module)
    return put


def test_missing(no_bind):
    no_bind(None)                         # (an import of it raises ImportError)
    with pytest.raises(RuntimeError, match="not found"):
        _lib.bind()
    with pytest.warns(RuntimeWarning, match="not found"):
        b = _lib.bind_or_none()
    assert b.kv_write(1, 2, 3) is None and b.kv_read() is None and b.tree_attn_q8(*range(16)) is None


@pytest.mark.parametrize("attr", [dict(), dict(torch="1.0"), dict(sizes=(1, 2, 3)), dict(torch="1.0", sizes=None)])
def test_stale(no_bind, attr):
    sizes = tuple(ctypes.sizeof(c) for c in (_lib.KvWriteArgs, _lib.KvReadArgs, _lib.AttnQ8Args))
    good = dict(torch=torch.__version__, sizes=sizes) | attr if attr else {}
    called = []
    no_bind(types.SimpleNamespace(init=lambda *a: called.append(a), **good))
    with pytest.raises(RuntimeError, match="built for"):
        _lib.bind()
    with pytest.warns(RuntimeWarning, match="built for"):
        assert _lib.bind_or_none() is _lib.NoBind
    assert not called


def test_present():
    b = _lib.bind()
    assert b is _lib.bind_or_none() and b.torch == torch.__version__


@pytest.mark.parametrize("error", ["status", "missing"])
def test_library_is_built_without_it(monkeypatch, tmp_path, error):
    lib, bind = str(tmp_path / "lib.so"), str(tmp_path / "_vnx_bind.so")
    for k, v in (("LIB_PATH", lib), ("BIND_PATH", bind), ("OBJ_DIR", str(tmp_path / "obj")), ("_hipcc", lambda: "hipcc")):
        monkeypatch.setattr(build, k, v)
    open(bind, "w").write("an older one")
    ran = []

    def run(cmd, **kw):
        ran.append(cmd[0])
        if cmd[0] != "hipcc":
            if error == "missing":
                raise FileNotFoundError("no compiler")
            return subprocess.CompletedProcess(cmd, 1, "", "no headers")
        open(cmd[cmd.index("-o") + 1], "w").write("x")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.warns(RuntimeWarning, match="is built, its Python binding is not"):
        assert build.build_library() == lib
    assert os.path.exists(lib) and not os.path.exists(bind) and len(ran) == len(build.sources()) + 2

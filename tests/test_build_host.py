"""What build() compiles, with the compilers replaced by a record of their commands."""

import os
import subprocess
import sys

import pytest


@pytest.fixture
def builder(monkeypatch, tmp_path):
    from cb200 import build as b
    ran = []

    def fake_run(cmd, **kw):
        ran.append(os.path.basename(cmd[0]))
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b.subprocess, "run", fake_run)
    monkeypatch.setattr(b, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(b, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "NATIVE_PATH", str(tmp_path / "native.so"))
    monkeypatch.setattr(b, "NATIVE_STAMP", str(tmp_path / "stamp"), raising=False)
    return b, ran


def _host(ran):
    return [c for c in ran if not c.startswith("nvcc")]


def test_without_torch_the_library_is_built_alone(builder, monkeypatch):
    b, ran = builder
    monkeypatch.setitem(sys.modules, "torch", None)
    assert b.build() == b.LIB_PATH
    assert len(ran) == len(b._sources()) + 1 and not _host(ran)
    assert not os.path.exists(b.NATIVE_PATH)
    ran.clear()
    b.build()
    assert ran == []


def test_the_torch_layer_follows_the_installed_torch(builder, monkeypatch):
    import torch
    b, ran = builder
    b.build()
    assert len(_host(ran)) == 1
    ran.clear()
    b.build()
    assert ran == []
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    b.build()
    assert len(ran) == 1 and len(_host(ran)) == 1  # the library need not be linked again
    ran.clear()
    b.build()
    assert ran == []

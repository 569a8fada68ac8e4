"""When the extension module is compiled again, and that no half of it is ever in place."""
from __future__ import annotations

import os
import types
from pathlib import Path

import pytest

pytest.importorskip("torch")
from sunnynet_b200 import build  # noqa: E402


@pytest.fixture
def made(tmp_path, monkeypatch):
    """A module that is newer than all it is made of; the compiler's calls."""
    include = tmp_path / "include"
    include.mkdir()
    (include / "sn_abi.h").write_text("")
    so = tmp_path / "_torch_calls.so"
    so.write_bytes(b"old")
    calls = []

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        calls.append(out)
        assert out != so and so.read_bytes() == b"old"
        out.write_bytes(b"new")
        return types.SimpleNamespace(returncode=run.rc, stderr="no")

    run.rc = 0
    monkeypatch.setattr(build, "INCLUDE", include)
    monkeypatch.setattr(build, "TORCH_CALLS", so)
    monkeypatch.setattr(build.subprocess, "run", run)
    late = max(p.stat().st_mtime for p in (build.CSRC / "torch_calls.cpp", Path(build.__file__))) + 1e6
    os.utime(so, (late, late))
    return types.SimpleNamespace(so=so, header=include / "sn_abi.h", calls=calls, run=run, late=late)


def test_compiled_again_when_a_signature_may_have_changed(made):
    build._build_torch_calls(False)
    assert not made.calls and made.so.read_bytes() == b"old"
    os.utime(made.header, (made.late + 5, made.late + 5))
    build._build_torch_calls(False)
    assert len(made.calls) == 1 and made.so.read_bytes() == b"new"
    assert sorted(p.name for p in made.so.parent.iterdir()) == ["_torch_calls.so", "include"]


def test_a_failed_build_leaves_the_old_module(made):
    made.run.rc = 1
    with pytest.raises(RuntimeError, match="failed"):
        build._build_torch_calls(True)
    assert made.calls and made.so.read_bytes() == b"old"
    assert sorted(p.name for p in made.so.parent.iterdir()) == ["_torch_calls.so", "include"]

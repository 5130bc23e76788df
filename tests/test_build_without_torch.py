"""Users of the C ABI build it where torch, or torch's g++, is not installed.  No compiler runs here."""
from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture
def build(monkeypatch):
    """vlx-tee_amd/build.py, which notes the commands instead of running them."""
    spec = importlib.util.spec_from_file_location("_build_under_test", ROOT / "vlx-tee_amd" / "build.py")
    B = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(B)
    B.commands = []
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **kw: B.commands.append(cmd))
    monkeypatch.setattr(B.os, "replace", lambda a, b: None)
    return B


def _outputs(B):
    return [Path(c[c.index("-o") + 1]).name for c in B.commands if "-c" not in c]


def test_everything_is_built_with_torch(build):
    pytest.importorskip("torch")
    assert build.build() == build.LIB
    assert _outputs(build) == ["libztcp_hip.so.tmp", "libztcp_hip_timers.so.tmp", "ztcp_capi_example.tmp", "_ztcp_torch.so.tmp"]


def test_the_library_is_built_without_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)   # "import torch" raises ImportError
    assert build.build() == build.LIB
    assert _outputs(build) == ["libztcp_hip.so.tmp", "libztcp_hip_timers.so.tmp", "ztcp_capi_example.tmp"]
    assert "torch binding left out" in capsys.readouterr().err


def test_the_binding_takes_rocm_and_a_compiler_where_they_are(build, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setenv("HIPCC", "/somewhere/rocm/bin/hipcc")
    monkeypatch.delenv("ROCM_PATH", raising=False)
    monkeypatch.delenv("CXX", raising=False)
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    build.build()
    assert build.commands[-1][0] == "/somewhere/rocm/bin/amdclang++"
    assert "/somewhere/rocm/include" in build.commands[-1] and "/opt/rocm/include" not in build.commands[-1]

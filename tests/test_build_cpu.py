"""The build where torch, or its headers, are missing: the library and the C++ check
program are built, and the Python module over torch's tensors is left out."""
import importlib.util
import os
import types

import pytest

from lutmac_amd import build as B


@pytest.mark.parametrize("torch", ["missing", "without headers"])
def test_build_without_torch(monkeypatch, capsys, tmp_path, torch):
    find = importlib.util.find_spec
    spec = None if torch == "missing" else types.SimpleNamespace(origin=str(tmp_path / "torch" / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec if name == "torch" else find(name, *a))
    run = []
    monkeypatch.setattr(B, "_run", lambda cmd, verbose: run.append(" ".join(cmd)))
    monkeypatch.setattr(os, "replace", lambda a, b: None)
    assert B.build(verbose=False) == B.LIB
    assert sum("-shared" in c and "liblutmac_hip.so" in c for c in run) == 1
    assert any("compat_smoke.cpp" in c for c in run) and not any("lmx_torch.cpp" in c for c in run)
    assert "_torch.so is left out" in capsys.readouterr().out


def test_build_with_torch(monkeypatch):
    run = []
    monkeypatch.setattr(B, "_run", lambda cmd, verbose: run.append(" ".join(cmd)))
    monkeypatch.setattr(os, "replace", lambda a, b: None)
    B.build(verbose=False)
    assert sum("lmx_torch.cpp" in c for c in run) == 1 and any("compat_smoke.cpp" in c for c in run)

"""The extension module asterq._calls is of one version of torch: with another it is built again, and not used until then."""
from __future__ import annotations

import types

import pytest
import torch

from asterq import _lib, build


def test_the_extension_is_not_used_with_another_torch(monkeypatch):
    module = _lib.quick_calls()
    if module is None:
        pytest.skip("asterq._calls is not built")
    monkeypatch.setattr(_lib, "_calls", None)
    assert _lib.quick_calls() is module
    monkeypatch.setattr(_lib, "_calls", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert _lib.quick_calls() is None


def test_the_extension_is_built_again_for_another_torch(monkeypatch):
    if not build.CALLS_PATH.exists():
        pytest.skip("asterq._calls is not built")
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        return types.SimpleNamespace(returncode=1, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "_stale", lambda target, deps: False)  # no source is newer
    build.build_calls()
    assert not runs
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(RuntimeError):
        build.build_calls()
    assert len(runs) == 1 and any("0.0.1" in word for word in runs[0])

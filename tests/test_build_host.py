"""What a change makes the build do again: the kernel library and the Python entry apart."""

from __future__ import annotations

import importlib.metadata

from musa_aiter import _build


def test_another_torch_rebuilds_the_python_entry_alone(monkeypatch):
    assert _build.build().ok and _build.is_built()
    ran = []
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0")
    monkeypatch.setattr(_build.subprocess, "run", lambda cmd, **k: ran.append(cmd) or Failed())
    assert not _build.is_built()
    assert not _build.build().ok
    assert len(ran) == 1 and str(_build.FRONT_SOURCE) in ran[0]


def test_nothing_changed_builds_nothing(monkeypatch):
    assert _build.build().ok
    monkeypatch.setattr(_build.subprocess, "run", None)
    assert _build.build().message == "up to date"


class Failed:
    returncode, stderr = 1, "not run"

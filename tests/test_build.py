"""CPU test of when the torch module of the 8-bit cache is built again (no compiler is run)."""

from __future__ import annotations

import importlib.util
import os
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent / "kitty-kv_b200"


def test_torch_module_is_built_again_for_another_torch(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("kitty_build", PKG / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    runs = []

    def compiler(cmd, check):
        runs.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("module")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    monkeypatch.setattr(build, "BUILD", tmp_path)
    module, src = tmp_path / "m.so", PKG / "csrc" / "kv8" / "kv8_torch.cpp"

    def count():
        build._torch_module(module, src, tmp_path / "lib.so", False)
        return len(runs)

    assert count() == 1 and module.exists() and count() == 1
    real = build.metadata.version
    monkeypatch.setattr(build.metadata, "version", lambda name: real(name) + ".other")
    assert count() == 2 and count() == 2
    monkeypatch.setattr(build.metadata, "version", real)
    assert count() == 3
    os.utime(module, (0, 0))                              # older than its source
    assert count() == 4 and count() == 4

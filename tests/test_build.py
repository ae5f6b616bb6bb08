"""When the torch binding is rebuilt (no compiler runs here)."""

import os
from pathlib import Path

import torch

from forma_b200 import build as fb


def test_binding_follows_its_sources_and_torch(monkeypatch, tmp_path):
    runs = []

    def compiler(cmd, check):
        runs.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("binding")

    monkeypatch.setattr(fb, "BIND", tmp_path / "_torch_bind.so")
    monkeypatch.setattr(fb, "OBJ", tmp_path / "_build")
    monkeypatch.setattr(fb.subprocess, "run", compiler)
    assert fb.build_bind() == tmp_path / "_torch_bind.so"
    assert len(runs) == 1
    fb.build_bind()
    assert len(runs) == 1  # up to date
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".next")
    fb.build_bind()
    assert len(runs) == 2  # built for another torch
    fb.build_bind()
    assert len(runs) == 2
    os.utime(fb.BIND, (0, 0))
    fb.build_bind()
    assert len(runs) == 3  # older than its sources
    fb.build_bind(force=True)
    assert len(runs) == 4

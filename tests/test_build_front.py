"""The library builds where the torch front end cannot: a user of the C ABI needs nvcc alone."""

from __future__ import annotations

import importlib.metadata
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

from leanstack_b200 import build as b

REPO = Path(__file__).resolve().parents[1]


def test_without_torch(tmp_path):
    code = (f"import sys; sys.modules['torch'] = None\n"
            f"from pathlib import Path\n"
            f"import leanstack_b200.build as b\n"
            f"b.needs_build = lambda defines=None: False\n"
            f"b.FRONT = Path({str(tmp_path)!r}) / '_torch_front.so'\n"
            f"print(b.build() == b.LIB)\n")
    res = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True,
                         env={**os.environ, "PYTHONPATH": str(REPO)})
    assert res.returncode == 0, res.stderr
    assert res.stdout.strip() == "True" and "no PyTorch" in res.stderr
    assert not list(tmp_path.iterdir())


def test_without_python_headers(tmp_path, monkeypatch, capsys):
    monkeypatch.setattr(b, "needs_build", lambda defines=None: False)
    monkeypatch.setattr(b, "FRONT", tmp_path / "_torch_front.so")
    paths = sysconfig.get_paths()
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {**paths, "include": str(tmp_path / "none")})
    assert b.build() == b.LIB
    assert "no Python's headers" in capsys.readouterr().err


def test_another_pytorch_needs_another_front(tmp_path, monkeypatch):
    monkeypatch.setattr(b, "FRONT", tmp_path / "_torch_front.so")
    monkeypatch.setattr(b, "FRONT_STAMP", tmp_path / "front_torch.txt", raising=False)
    version = importlib.metadata.version("torch")
    (tmp_path / "front_torch.txt").write_text(version + "\n")
    (tmp_path / "_torch_front.so").touch()
    assert not b.needs_front()
    (tmp_path / "front_torch.txt").write_text("0.0.1\n")
    assert b.needs_front()

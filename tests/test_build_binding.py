"""When the torch binding of the paged calls is built, with stand-ins for the installed torch."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import REPO


def stand_in(folder, version: str, *, cuda: bool):
    root = folder / "torch"
    (root / "lib").mkdir(parents=True)
    (root / "__init__.py").write_text("raise ImportError('only looked up')\n")
    (root / "version.py").write_text(f"__version__ = '{version}'\ncuda = {'12.8' if cuda else None!r}\n")
    if cuda:
        (root / "lib" / "libc10_cuda.so").write_text("")
    return folder


def up_to_date(folder, binding) -> bool:
    """calls_up_to_date() of a process that finds the stand-in, for the binding at that path."""
    code = f"from pathlib import Path; from llaccel_b200 import build as B; B.CALLS = Path({str(binding)!r}); print(B.calls_up_to_date())"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=REPO,
                       env=dict(os.environ, PYTHONPATH=f"{folder}{os.pathsep}{REPO}"))
    assert r.returncode == 0, r.stderr
    return r.stdout.strip() == "True"


def test_a_torch_without_cuda_needs_no_binding(tmp_path):
    assert up_to_date(stand_in(tmp_path / "cpu", "2.11.0+cpu", cuda=False), tmp_path / "none.so")
    assert not up_to_date(stand_in(tmp_path / "gpu", "2.11.0+cu128", cuda=True), tmp_path / "none.so")


def test_another_torch_needs_another_binding(tmp_path):
    from llaccel_b200 import build
    build.build()
    if not build.CALLS.exists():
        pytest.skip("no binding here")
    assert build.calls_up_to_date()
    assert not up_to_date(stand_in(tmp_path, "2.99.0+cu130", cuda=True), build.CALLS)

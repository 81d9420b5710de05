"""The C++ calls from torch are an extra: the C library builds without torch,
and the Python calls serve where that extra is missing or does not load."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

PKG = Path(__file__).resolve().parent.parent / "ndtensors-rs_b200"


def planned(*args):
    return subprocess.run(["make", "-n", "-B", "-C", str(PKG), *args], capture_output=True, text=True)


def test_the_c_library_builds_without_torch():
    run = planned(f"PYTHON={sys.executable} -S")  # (no site-packages)
    assert run.returncode == 0, run.stderr
    assert "libndtensors_capi.so" in run.stdout and "torch_calls" not in run.stdout


def test_the_calls_are_built_where_torch_is():
    run = planned(f"PYTHON={sys.executable}")
    assert run.returncode == 0, run.stderr
    assert "csrc/torch_calls.cpp" in run.stdout


def test_the_calls_are_built_again_for_another_torch():
    run = subprocess.run(["make", "-n", "-C", str(PKG), f"PYTHON={sys.executable}", "TORCH_VERSION=0.0.0"],
                         capture_output=True, text=True)
    assert run.returncode == 0 and "csrc/torch_calls.cpp" in run.stdout


@pytest.mark.parametrize("kind", ["missing", "broken"])
def test_python_serves_without_them(ndt, tmp_path, kind):
    from ndtensors_b200 import _model

    path = tmp_path / "ndt_torch_calls.so"
    if kind == "broken":
        path.write_bytes(b"not a library")
    with pytest.warns(RuntimeWarning, match="ndt_torch_calls"):
        calls = _model._load_calls(path)
    for name in ("embedding", "torch_embedding", "scaled_linear", "torch_scaled_linear"):
        assert getattr(calls, name)(None, None, None, None) is None


def test_they_load_here(ndt):
    from ndtensors_b200 import _model

    assert type(_model.calls).__name__ == "module"

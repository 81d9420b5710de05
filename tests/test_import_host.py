"""The package without torch: everything but the torch operators is there."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent / "ndtensors-rs_b200"


def run(code):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=PKG)


def test_import_star_without_torch():
    r = run("import sys; sys.modules['torch'] = None\nfrom ndtensors_b200 import *\nassert callable(contract) and callable(TensorF64.zeros)")
    assert r.returncode == 0, r.stderr


def test_a_torch_operator_without_torch_says_so():
    r = run("import sys; sys.modules['torch'] = None\nimport ndtensors_b200 as ndt\n"
            "try:\n    ndt.embedding\nexcept ImportError as e:\n    assert 'torch' in str(e)\nelse:\n    raise SystemExit(1)")
    assert r.returncode == 0, r.stderr

"""The dense operators beside torch, in a process that imports torch first."""

import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_calls_beside_torch() -> None:
    if importlib.util.find_spec("torch") is None:  # (not imported here: it brings a HIP runtime of its own)
        pytest.skip("no torch")
    r = subprocess.run([sys.executable, "-u", str(Path(__file__).with_name("dense_torch_calls.py"))], capture_output=True,
                       text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.count("passed") == 5, r.stdout + r.stderr

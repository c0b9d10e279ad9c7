"""The serving example runs, and its answers are those of the contiguous attention."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "serve_shared_prefix.py"


@pytest.mark.parametrize("args", [[], ["--conversations", "3", "--prefix", "77", "--steps", "40", "--kv-heads", "8"]])
def test_serve_shared_prefix(cuda, args):
    r = subprocess.run([sys.executable, str(EXAMPLE), "--check", *args], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "tokens/s" in r.stdout and "largest relative difference" in r.stdout

"""A program whose first use of the library is a captured one: few rows, one wave of small tiles, CTA pairs."""
import subprocess
import sys
from pathlib import Path

import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 70, 4000])
def test_first_calls_may_be_captured(hom, rows):
    script = Path(__file__).with_name("first_call_captured.py")
    run = subprocess.run([sys.executable, str(script), str(rows)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr

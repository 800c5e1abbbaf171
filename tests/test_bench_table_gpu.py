"""The engine-style table at a context depth: `bench.py --table -d` runs every layer with its attention half."""
import os
import re
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_table_with_a_context_depth():
    r = subprocess.run([sys.executable, "bench.py", "--table", "--layers", "2", "-p", "64,300", "-n", "4", "-r", "2", "-d", "0,700"], cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    rows = re.findall(r"\| (\S.*?) \| (pp64|pp300|tg4)( @ d\d+)? \| ([0-9.]+) ", r.stdout)
    assert [(t, d.strip()) for _, t, d, _ in rows] == [("pp64", ""), ("pp300", ""), ("tg4", "")] + [(t, f"@ d{d}") for d in (0, 700) for t in ("pp64", "pp300", "tg4")]
    assert all(float(x) > 0 for *_, x in rows)

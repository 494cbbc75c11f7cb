"""bench.py --impl reference answers for the reference or not at all: where its code is absent, one line says so."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_unavailable_without_the_reference(tmp_path):
    if (ROOT / "oracle" / "_ref" / "libref_host.so").exists():
        pytest.skip("compiled reference helpers present")
    run = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--gpus", "1", "--steps", "1", "--warmup", "1"], cwd=ROOT,
                         env={**os.environ, "REF": str(tmp_path)}, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    lines = run.stdout.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line

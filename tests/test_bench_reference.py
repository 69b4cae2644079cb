"""The bench's reference arm without the reference."""
from __future__ import annotations

import json
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_reference_arm_without_the_reference_is_unavailable():
    """Its line says so, and no other code is timed under the reference's name."""
    run = """
import sys, oracle, bench
from pathlib import Path
oracle.REF_ORACLE_LIB = Path("/nonexistent")
oracle.reference_case = None
sys.argv = ["bench.py", "--impl", "reference", "--steps", "2", "--warmup", "3"]
sys.exit(bench.main())
"""
    done = subprocess.run([sys.executable, "-c", run], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    lines = [json.loads(x) for x in done.stdout.splitlines()]
    assert len(lines) == 1 and lines[0]["impl"] == "reference"
    assert lines[0]["unavailable"] and "value" not in lines[0]

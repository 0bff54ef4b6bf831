"""bench.py --impl reference without the reference's kernels: it says so, and no other implementation's figure stands in their place."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("workload", ["decode", "prefill"])
def test_an_absent_reference_is_called_unavailable(workload):
    sys.path.insert(0, ROOT)
    from oracle import refptx
    if refptx.available():
        pytest.skip("the reference's kernels are built here")
    r = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--gpus", "1", "--steps", "3", "--warmup", "3", "--workload", workload],
                       cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout)
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line

"""The benchmark's reference arm must answer on any machine: one JSON line, exit code 0."""

import json
import os
import subprocess
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_reference_arm_reports_unavailable():
    p = subprocess.run([sys.executable, os.path.join(REPO, "bench.py"), "--impl", "reference", "--gpus", "1",
                        "--steps", "1", "--warmup", "3"], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-500:]
    line = [l for l in p.stdout.splitlines() if l.startswith("{")][-1]
    d = json.loads(line)
    assert d["impl"] == "reference" and isinstance(d["unavailable"], str) and d["unavailable"]


def test_the_line_names_the_type_of_the_linears():
    sys.path.insert(0, REPO)
    import bench
    assert bench.compute_type(None) == "bf16" and bench.compute_type("fp8") == "fp8-weights/bf16-activations"
    assert bench.compute_type("nvfp4").startswith("nvfp4-") and bench.compute_type("mxfp4").startswith("mxfp4-")

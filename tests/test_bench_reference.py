"""bench.py --impl reference runs the reference's own code, or says that it cannot."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_restatement_does_not_stand_in_for_the_reference():
    from oracle import gwo
    if gwo.load("ref") is not None:
        pytest.skip("oracle/_ref is built")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--impl", "reference", "--steps", "1", "--warmup", "3"], capture_output=True, text=True,
                       timeout=120, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-400:]
    line = json.loads(r.stdout.strip().splitlines()[-1])
    assert line["impl"] == "reference" and "value" not in line and "oracle/_ref" in line["unavailable"]

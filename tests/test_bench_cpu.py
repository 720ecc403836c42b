"""bench.py's reference arm on a machine without the host framework."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def _missing():
    from mira_b200.hostfw import import_mira
    try:
        import_mira()
    except ImportError:
        return True
    return False


@pytest.mark.skipif(not _missing(), reason="the MIRA host framework is installed")
@pytest.mark.parametrize("workload", ["resnet18", "decode"])
def test_reference_arm_says_why_it_cannot_run(workload):
    run = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--workload", workload, "--steps", "2", "--warmup", "1"],
                         cwd=ROOT, env=dict(os.environ), capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    line = json.loads(run.stdout)
    assert set(line) == {"impl", "unavailable"} and line["impl"] == "reference" and "mira" in line["unavailable"]
    assert "\n" not in line["unavailable"]

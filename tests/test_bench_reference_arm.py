"""bench.py --impl reference: the reference's path alone, none of this package's code in its process."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUN = """
import runpy, sys
sys.argv = ["bench.py", "--impl", "reference", "--steps", "1", "--warmup", "3", *{more}]
try:
    runpy.run_path("bench.py", run_name="__main__")
except SystemExit as e:
    assert not e.code, e.code
assert not [m for m in sys.modules if m.split(".")[0] == "pla_b200"], "package imported"
assert "libpla_b200" not in open("/proc/self/maps").read(), "library mapped"
"""


@pytest.mark.parametrize("more", [["--grid", "512"], ["--workload", "dw_cfg1"], ["--workload", "dwln_cfg4"]], ids=["default", "depthwise", "layernorm"])
def test_reference_arm_loads_nothing_of_this_package(more):
    r = subprocess.run([sys.executable, "-c", RUN.format(more=more)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert json.loads(r.stdout.strip().splitlines()[-1])["impl"] == "reference"

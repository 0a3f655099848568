"""bench.py's fp8 workload with attention as its compute: the layer-wise restore
with the paged-cache operators on a second stream, end to end."""

import json
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def test_fp8_workload_with_attention():
    p = subprocess.run([sys.executable, str(ROOT / "bench.py"), "--workload", "llama8b_fp8_evict", "--fp8-requests", "2",
                        "--fp8-pool-gb", "4", "--fp8-compute", "attention"], capture_output=True, text=True, timeout=600,
                       cwd=ROOT)
    assert p.returncode == 0, p.stderr[-2000:]
    line = json.loads(p.stdout.strip().splitlines()[-1])
    assert line["engine"]["load_failures"] == 0 and line["layerwise_overlap"]["hit_blocks"] > 0
    assert "attention" in line["config"]["compute_ms_per_layer"]

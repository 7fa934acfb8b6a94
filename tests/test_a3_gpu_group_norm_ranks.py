"""PartitionedGAT(norm="group") as it runs on a node: the fused operators, over RCCL on one rank and over gloo on two
ranks that share the card (tests/rehearse_group_norm_gpu.py).  The children start before this process touches the GPU:
the file name sorts behind test_a2."""
import os
import subprocess
import sys

import pytest

from test_a1_gpu_rccl_world1 import _env
from test_a2_gpu_gloo_world2 import _launch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu
SCRIPT = os.path.join(ROOT, "tests", "rehearse_group_norm_gpu.py")


@pytest.mark.parametrize("how", ["nccl", "gloo"])
def test_partitioned_group_norm_network(how):
    if how == "nccl":
        r = subprocess.run([sys.executable, SCRIPT, how], env=_env(29698), capture_output=True, text=True, timeout=110)
    else:
        r = _launch(29699, [SCRIPT, how], 110)
    lines = [ln for ln in r.stdout.splitlines() if ln.startswith(("ok", "FAILED"))]
    if r.returncode != 0 and not lines and "init_process_group" in r.stderr:
        pytest.skip(f"{how} group could not be created here: " + r.stderr[-400:])
    assert r.returncode == 0 and len(lines) == 3 and all(ln.startswith("ok") for ln in lines), \
        r.stdout[-2000:] + r.stderr[-3000:]

"""Where the operators on the direct xGMI all-reduce find and leave their tensors, with several rank
processes mapped onto the one GPU (tests/xgmi_ops_buffers_worker.py)."""

import json
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

WORKER = Path(__file__).resolve().parent / "xgmi_ops_buffers_worker.py"


def _ranks(world, *args):
    from network_operator_amd.parallel.xgmi_comm import spawn_ranks

    procs, outs = spawn_ranks(world, [sys.executable, str(WORKER), *args], timeout=100)
    assert all(p.returncode == 0 for p in procs), "\n".join(o[-2000:] for o in outs)
    return [json.loads(next(x[7:] for x in o.splitlines() if x.startswith("RESULT "))) for o in outs]


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 3])
def test_a_residual_in_the_output_buffer_keeps_its_values(cuda_device, world):
    for r in _ranks(world, "residual"):
        assert len(r) == 8 and not any(r.values()), r

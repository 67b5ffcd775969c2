"""The operators on the direct xGMI all-reduce (XgmiAllReduce.all_reduce_norm, ShardedAdamW), with
several rank processes mapped onto the one GPU (tests/xgmi_ops_worker.py)."""

import json
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

WORKER = Path(__file__).resolve().parent / "xgmi_ops_worker.py"


def _ranks(world, mode):
    from network_operator_amd.parallel.xgmi_comm import spawn_ranks

    procs, outs = spawn_ranks(world, [sys.executable, str(WORKER), mode], timeout=100)
    assert all(p.returncode == 0 for p in procs), "\n".join(o[-2000:] for o in outs)
    return [json.loads(next(x[7:] for x in o.splitlines() if x.startswith("RESULT "))) for o in outs]


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 2, 3])
def test_all_reduce_norm_equals_the_norm_of_all_partial_sums(cuda_device, world):
    for r in _ranks(world, "norm"):
        assert len(r) == 8 and not any(r.values()), r


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 3])
def test_sharded_adamw_equals_adamw_on_whole_tensors(cuda_device, world):
    for r in _ranks(world, "adamw"):
        # the norm is added up in another order: its last bit may turn the factor's, a 2^-24th of a step,
        # and with it a rounding of a parameter here and there by one step of bf16 (2^-6 between 2 and 4)
        assert r["far"] <= 2 ** -6 and r["norm_off"] <= 4 * 2 ** -24, r
        assert r["infinite_norm"] and r["kept"] and r["alike"], r


def test_sharded_adamw_refuses():
    from network_operator_amd.parallel.sharded_adamw import ShardedAdamW

    class Comm:
        rank, world, device = 0, 2, torch.device("cpu")

    with pytest.raises(ValueError, match="no parameters"):
        ShardedAdamW(Comm(), [], lr=1e-3)
    for bad in (torch.zeros(8), torch.zeros(8, 4, dtype=torch.bfloat16).t(), torch.zeros(8, dtype=torch.bfloat16, device="meta")):
        with pytest.raises(ValueError, match="contiguous bfloat16"):
            ShardedAdamW(Comm(), [bad], lr=1e-3)
    with pytest.raises(ValueError, match="max_norm"):
        ShardedAdamW(Comm(), [torch.zeros(8, dtype=torch.bfloat16)], lr=1e-3, max_norm=-1.0)

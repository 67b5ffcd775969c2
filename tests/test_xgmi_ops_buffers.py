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


def test_a_refused_norm_does_not_leave_its_peers_at_the_barrier(monkeypatch):
    """A launch that is refused between the two barriers of the one-shot norm: the rank takes part in both."""
    from network_operator_amd.parallel import xgmi_comm

    comm = object.__new__(xgmi_comm.XgmiAllReduce)
    comm.rank, comm.world, comm.capacity, comm.device = 0, 2, 1024, torch.device("cpu")
    comm.inp, comm.out, comm.peer_in = torch.zeros(1024, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), [1, 2]
    seen = []

    def refuse(*args):
        seen.append("launch")
        raise ValueError("an output overlaps another tensor of the call")

    monkeypatch.setattr(comm, "_sync_and_wait", lambda stream: seen.append("barrier"))
    monkeypatch.setattr(xgmi_comm.N, "_arguments", lambda *args: ([0, 0],))
    monkeypatch.setattr(xgmi_comm.N, "_launch", refuse)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: None)
    with pytest.raises(ValueError, match="overlaps"):
        comm.all_reduce_norm(torch.ones(16), torch.zeros(4, 16, dtype=torch.bfloat16), algo="one_shot")
    assert seen == ["barrier", "launch", "barrier"]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("world", [1, 3])
def test_sharded_states_are_those_of_the_parameters_parts(cuda_device, world, bits):
    for r in _ranks(world, "pieces", str(bits)):
        assert not any(r.values()), r


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 2])
def test_an_overflowed_step_after_loading_keeps_the_loaded_parameters(cuda_device, world):
    for r in _ranks(world, "load"):
        assert not any(r.values()), r


@pytest.mark.gpu
def test_a_device_without_an_index_is_the_current_one(cuda_device):
    assert _ranks(1, "device") == [{"device": 0}]


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 3])
def test_sharded_steps_are_clipped_averaged_and_decayed(cuda_device, world):
    """In units of u = 2^-24.  A rank's norm is off by 2 u (the factor 1 / ranks, a rounding), the factor by
    one more, the other side's by 1: with a rounding a side, gradients x differ by 6 u.  M is the largest |x| so
    far, c_k = 1 - 0.9^k.  m: d_k <= 0.9 d_(k-1) + 0.1 * 6 + 2 sides * 2 c_k, so d_1..3 = 1, 2.3, 3.8 (of M); v (of
    M^2): 0.001 * (14 + 4 k) a step, 0.07.  The update, at most 1.73 lr: m's share d_k / c_k / 0.58 = 24, sqrt(v)'s
    (14 + 12) / 2 + 2 = 15 and 12 roundings on the way, (15 + 12) * 1.73 = 47, in units of lr; 4 u a step of the
    master's own magnitude.  Three steps: 3 * (4 + 24 + 47), with lr added to the magnitude."""
    rows = _ranks(world, "clip")
    for r in rows:
        assert r["exp_avg"] <= 4 and r["exp_avg_sq"] <= 0.1 and r["master"] <= 225 and r["parameters"] == 0, r
    assert sum(r["checked"] for r in rows) == 33 * 5 + 1000 + 7 + 64 * 64, rows


def test_sharded_adamw_refuses_parameters_that_share_memory():
    """A tied weight given twice: its gradient would count twice in the norm, and two masters would drift apart."""
    from network_operator_amd.parallel.sharded_adamw import ShardedAdamW

    class Comm:
        rank, world, device = 0, 2, torch.device("cpu")

    p = torch.zeros(16, dtype=torch.bfloat16)
    for pair in ([p, p], [p[:9], p[8:]]):
        with pytest.raises(ValueError, match="share memory"):
            ShardedAdamW(Comm(), pair, lr=1e-3)

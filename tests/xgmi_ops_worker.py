"""Rank process of tests/test_xgmi_ops.py: the operators on the direct xGMI all-reduce, all ranks
on GPU 0.

    RANK=r WORLD_SIZE=n NETOP_INIT_FILE=... python xgmi_ops_worker.py norm | adamw
"""

import faulthandler
import json
import os
import sys

import torch
import torch.distributed as dist

from network_operator_amd.ops import norm
from network_operator_amd.parallel.sharded_adamw import ShardedAdamW
from network_operator_amd.parallel.xgmi_comm import XgmiAllReduce

faulthandler.dump_traceback_later(float(os.environ.get("NETOP_RANK_HANG_S", "90")), exit=True)
DEV = torch.device("cuda", 0)


def _partial(rank, rows, cols, seed):
    g = torch.Generator().manual_seed(100 * seed + rank)
    return (torch.randn(rows, cols, generator=g) * 0.5).bfloat16()


def run_norm(rank, world):
    """one_shot equals add_rms_norm over the same partial sums in rank order, bit for bit; the
    two-shot variants equal it over the sum rounded to bf16; buffers reused, several shapes."""
    comm = XgmiAllReduce(1 << 20, device=DEV)
    wrong = {}
    for i, (rows, cols, algo, kind) in enumerate([
            (4, 1024, "one_shot", "same"), (7, 129, "auto", "same"), (16, 2048, "one_shot", "row"), (3, 1000, "auto", "group"),
            (24, 2048, "two_shot", "same"), (24, 2048, "two_shot_push", "row"), (1, 64, "auto", "same"), (0, 64, "auto", "same")]):
        parts = [_partial(r, rows, cols, i).to(DEV) for r in range(world)]
        res = _partial(99, rows, cols, i).to(DEV)
        w = (1 + 0.1 * _partial(98, 1, cols, i).float()[0]).to(DEV)
        got, want = ([torch.empty(rows, cols, dtype=torch.bfloat16 if kind == "same" else torch.float8_e4m3fn, device=DEV),
                      torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV), torch.empty(rows, device=DEV),
                      None if kind == "same" else torch.empty((rows,) if kind == "row" else (rows, -(-cols // 128)), device=DEV)]
                     for _ in range(2))
        comm.input(rows * cols).view(rows, cols).copy_(parts[rank])
        comm.all_reduce_norm(w, got[0], residual=res, residual_out=got[1], rstd=got[2], scales=got[3], algo=algo)
        if "two" in algo:
            total = torch.zeros(rows, cols, device=DEV)
            for p in parts:
                total += p.float()
            parts = [total.bfloat16()]
        norm.add_rms_norm(parts, w, want[0], residual=res, residual_out=want[1], rstd=want[2], scales=want[3])
        wrong[f"{i} {rows}x{cols} {algo} {kind}"] = sum(
            int((a.view(torch.uint8) != b.view(torch.uint8)).sum()) for a, b in zip(got, want) if a is not None and a.numel())
    for what, out in (("fp32", torch.empty(4, 64, device=DEV)), ("in the input buffer", comm.input(256).view(4, 64)),
                      ("too large", torch.empty(1 << 14, 64, dtype=torch.bfloat16, device=DEV))):
        try:
            comm.all_reduce_norm(w, out)
            wrong[what + " accepted"] = 1
        except ValueError:
            pass
    comm.close()
    return wrong


def run_adamw(rank, world):
    """Three sharded steps against the same steps on whole tensors (ops/adamw.py) from the summed
    gradients, parameters that end anywhere in a rank's chunk; a step of an infinite gradient."""
    from network_operator_amd.ops import adamw

    sizes = [(33, 5), (1000,), (7,), (64, 64)]
    g = torch.Generator().manual_seed(3)
    start = [(torch.randn(s, generator=g)).bfloat16().to(DEV) for s in sizes]
    params = [torch.nn.Parameter(p.clone()) for p in start]
    ref = [p.clone() for p in start]
    comm = XgmiAllReduce(1 << 20, device=DEV)
    opt = ShardedAdamW(comm, params, lr=1e-2, weight_decay=0.1, max_norm=0.5)
    whole = adamw.AdamW(ref, lr=1e-2, weight_decay=0.1)
    norm_off = 0.0
    for step in (1, 2, 3):
        sums = [torch.zeros(s, device=DEV) for s in sizes]
        for r in range(world):
            gr = torch.Generator().manual_seed(1000 * step + r)
            for p, s, total in zip(params, sizes, sums):
                x = torch.randn(s, generator=gr).bfloat16().to(DEV)
                total += x.float()
                if r == rank:
                    p.grad = x
        if step == 2:  # a parameter no rank has a gradient for
            params[2].grad = None
            sums[2].zero_()
        got = opt.step(step)
        grads = [t.bfloat16() for t in sums]
        total, coef = torch.empty(1, device=DEV), torch.empty(1, device=DEV)
        adamw.grad_norm(grads, total, coef=coef, max_norm=0.5, scale=1 / world)
        whole.step(grads, step=step, coef=coef)
        norm_off = max(norm_off, abs(got / float(total) - 1))
    same = [torch.equal(p.detach(), q) for p, q in zip(params, ref)]
    far = max(float((p.detach().float() - q.float()).abs().max()) for p, q in zip(params, ref))
    before = [p.detach().clone() for p in params]
    for p in params:
        p.grad = torch.zeros_like(p)
    if rank == world - 1:
        params[0].grad[0, 0] = float("inf")
    bad = opt.step(4)
    kept = all(torch.equal(p.detach(), b) for p, b in zip(params, before))
    gathered = [None] * world
    dist.all_gather_object(gathered, [p.detach().cpu() for p in params])
    alike = all(torch.equal(a, b) for other in gathered for a, b in zip(other, gathered[0]))
    comm.close()
    return {"same": sum(same), "far": far, "norm_off": norm_off, "infinite_norm": bad == float("inf"), "kept": kept,
            "alike": alike}


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo", init_method=f"file://{os.environ['NETOP_INIT_FILE']}", rank=rank, world_size=world)
    torch.cuda.set_device(DEV)
    print("RESULT " + json.dumps({"norm": run_norm, "adamw": run_adamw}[sys.argv[1]](rank, world)), flush=True)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()

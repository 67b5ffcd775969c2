"""Rank process of tests/test_xgmi_ops_buffers.py: where the operators' tensors lie in the symmetric
buffers, and how the sharded optimizer cuts its states; all ranks on GPU 0.

    RANK=r WORLD_SIZE=n NETOP_INIT_FILE=... python xgmi_ops_buffers_worker.py MODE [ARGUMENT]
"""

import faulthandler
import json
import os
import sys

import torch
import torch.distributed as dist

from network_operator_amd.ops import adamw, norm
from network_operator_amd.parallel.sharded_adamw import ShardedAdamW
from network_operator_amd.parallel.xgmi_comm import XgmiAllReduce

faulthandler.dump_traceback_later(float(os.environ.get("NETOP_RANK_HANG_S", "90")), exit=True)
DEV = torch.device("cuda", 0)


def _bf16(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).bfloat16().to(DEV)


def _differ(a, b):
    return a.shape != b.shape or int((a.contiguous().view(torch.uint8) != b.contiguous().view(torch.uint8)).sum())


def run_residual(rank, world):
    """A residual or weight in the output buffer, which the two-shot variants write: the norm is that of
    the values it had.  On every rank, or on one alone."""
    rows, cols = 2112, 1024  # 4.1 MiB: "auto" takes two shots
    n = rows * cols
    comm = XgmiAllReduce(16 << 20, device=DEV)
    w = (1 + 0.1 * _bf16(cols, 1).float()).bfloat16()
    wrong = {}
    for i, (algo, where) in enumerate([("two_shot", "residual"), ("two_shot_push", "residual"), ("auto", "residual"),
                                       ("one_shot", "residual"), ("two_shot", "rank 0"), ("two_shot", "in place"),
                                       ("two_shot", "weight"), ("two_shot", "behind the message")]):
        parts = [_bf16((rows, cols), 100 * i + r, 0.5) for r in range(world)]
        res = _bf16((rows, cols), 100 * i + 99)
        out, want, h, want_h = (torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV) for _ in range(4))
        residual, weight = res, w
        if where == "weight":
            weight = comm.output(cols)
            weight.copy_(w)
        elif where == "behind the message":
            residual = comm.output(2 * n)[n:].view(rows, cols)
            residual.copy_(res)
        elif where != "rank 0" or rank == 0:
            residual = comm.output(n).view(rows, cols)
            residual.copy_(res)
            h = residual if where == "in place" else h
        comm.input(n).view(rows, cols).copy_(parts[rank])
        comm.all_reduce_norm(weight, out, residual=residual, residual_out=h, algo=algo)
        total = torch.zeros(rows, cols, device=DEV)
        for p in parts:
            total += p.float()
        norm.add_rms_norm(parts if algo == "one_shot" or world == 1 else [total.bfloat16()], w, want, residual=res,
                          residual_out=want_h)
        wrong[f"{algo} {where}"] = _differ(out, want) + _differ(h, want_h)
    comm.close()
    return wrong


def _sums(sizes, step, rank, world, params):
    """This rank's gradients into ``params``; the gradients of all ranks, summed in rank order in fp32 and
    rounded to bf16 as the reduce-scatter does."""
    sums = [torch.zeros(s, device=DEV) for s in sizes]
    for r in range(world):
        for k, (p, s) in enumerate(zip(params, sizes)):
            x = _bf16(s, 10000 * step + 100 * k + r, 0.1)
            sums[k] += x.float()
            if r == rank:
                p.grad = x
    return [t.bfloat16() for t in sums]


def run_pieces(rank, world, bits):
    """The states are those of AdamW over the parts of the parameters that lie in this rank's chunk, each
    a tensor of its own: bit for bit, three steps.  Small values beside large ones, a rank without any."""
    wrong = {}
    for i, sizes in enumerate([[(33, 5), (1000,), (7,), (64, 64), (300,)], [(9,)]]):
        scale = [0.02, 1.0, 1e-3, 0.02, 1e-3]
        comm = XgmiAllReduce(1 << 20, device=DEV)
        params = [torch.nn.Parameter(_bf16(s, k, scale[k])) for k, s in enumerate(sizes)]
        opt = ShardedAdamW(comm, params, lr=1e-2, weight_decay=0.1, state_bits=int(bits), seed=5)
        chunk = opt.numel // world
        lo, hi = rank * chunk, (rank + 1) * chunk
        cut = [(k, max(at, lo) - at, min(at + p.numel(), hi) - at) for k, (p, at) in enumerate(zip(params, opt.offsets))
               if max(at, lo) < min(at + p.numel(), hi)]

        def parts(tensors):
            return [tensors[k].detach().reshape(-1)[a:b] for k, a, b in cut]

        mine = [t.clone() for t in parts(params)]
        ref = adamw.AdamW(mine, lr=1e-2, weight_decay=0.1, state_bits=int(bits), seed=(5 + 0x9E3779B1 * rank) % (1 << 32)) if cut else None
        coef = torch.full((1,), 1 / world, device=DEV)
        for step in (1, 2, 3):
            sums = _sums(sizes, step, rank, world, params)
            for t in (sums[-1], params[-1].grad):  # a small gradient beside the others'
                t.mul_(2.0 ** -12)
            opt.step(step)
            if ref:
                ref.step(parts(sums), step=step, coef=coef)
        wrong[f"{i} parameters"] = sum(_differ(a, b) for a, b in zip(parts(params), mine))
        want = ref.state_dict() if ref else {}
        for k, t in opt.state_dict().items():
            if k in want and isinstance(t, torch.Tensor):
                wrong[f"{i} {k}"] = int(_differ(t, want[k]))
        gathered = [None] * world
        dist.all_gather_object(gathered, [p.detach().cpu() for p in params])
        wrong[f"{i} ranks differ"] = sum(_differ(a, b) for other in gathered for a, b in zip(other, gathered[0]))
        comm.close()
    return wrong


def run_clip(rank, world):
    """Clipped and averaged steps against the same steps on whole tensors: masters and moments by how far
    they are off in units of 2^-24 of what goes into them, parameters by their masters' roundings."""
    sizes = [(33, 5), (1000,), (7,), (64, 64)]
    params = [torch.nn.Parameter(_bf16(s, k)) for k, s in enumerate(sizes)]
    comm = XgmiAllReduce(1 << 20, device=DEV)
    opt = ShardedAdamW(comm, params, lr=1e-2, weight_decay=0.1, max_norm=0.5)
    whole = adamw.AdamW([p.detach().clone() for p in params], lr=1e-2, weight_decay=0.1)
    total, coef = torch.empty(1, device=DEV), torch.empty(1, device=DEV)
    mags = [torch.zeros(s, device=DEV) for s in sizes]
    for step in (1, 2, 3):
        sums = _sums(sizes, step, rank, world, params)
        opt.step(step)
        adamw.grad_norm(sums, total, coef=coef, max_norm=0.5, scale=1 / world)
        whole.step(sums, step=step, coef=coef)
        for m, s in zip(mags, sums):
            m.copy_(torch.maximum(m, s.float().abs() * coef))
    lo, hi = opt.mine.start, opt.mine.stop
    off, checked = dict(master=0.0, exp_avg=0.0, exp_avg_sq=0.0, parameters=0), 0
    at = 0  # in this rank's states
    for k, (p, start) in enumerate(zip(params, opt.offsets)):
        a, b = max(start, lo), min(start + p.numel(), hi)
        if a >= b:
            continue
        here, there = slice(at, at + b - a), slice(whole.offsets[k] + a - start, whole.offsets[k] + b - start)
        mag = mags[k].reshape(-1)[a - start:b - start]
        for name, scale in (("master", whole.master[there].abs() + 0.01), ("exp_avg", mag), ("exp_avg_sq", mag * mag)):
            x, y = getattr(opt.opt, name)[here], getattr(whole, name)[there]
            off[name] = max(off[name], float(((x - y).abs() / scale.clamp(min=1e-30)).max()) * 2 ** 24)
        off["parameters"] += _differ(p.detach().reshape(-1)[a - start:b - start], opt.opt.master[here].bfloat16())
        checked += b - a
        at += -(-(b - a) // 256) * 256
    comm.close()
    return dict(off, checked=checked)


def run_load(rank, world):
    """States and parameters loaded into an optimizer that was made from others: a step of an infinite
    norm leaves the parameters as they are, and the next one goes on from the loaded states."""
    sizes = [(40, 9), (511,)]

    def made(seed):
        params = [torch.nn.Parameter(_bf16(s, seed + k)) for k, s in enumerate(sizes)]
        return params, ShardedAdamW(comm, params, lr=1e-2, weight_decay=0.1)

    comm = XgmiAllReduce(1 << 20, device=DEV)
    old, a = made(0)
    for step in (1, 2):
        _sums(sizes, step, rank, world, old)
        a.step(step)
    saved = {k: t.clone() if isinstance(t, torch.Tensor) else t for k, t in a.state_dict().items()}
    new, b = made(50)
    with torch.no_grad():
        for p, q in zip(new, old):
            p.copy_(q)
    b.load_state_dict(saved)
    for p in new:
        p.grad = torch.zeros_like(p)
    new[1].grad[0] = float("inf")
    bad = b.step(3)
    got = {"norm is finite": int(bad != float("inf")), "kept": sum(_differ(p.detach(), q.detach()) for p, q in zip(new, old))}
    _sums(sizes, 3, rank, world, old)
    a.step(3)
    _sums(sizes, 3, rank, world, new)
    b.step(3)
    got["next"] = sum(_differ(p.detach(), q.detach()) for p, q in zip(new, old))
    comm.close()
    return got


def run_device(rank, world):
    """A communicator on "cuda" is one on the current device, and takes that device's parameters."""
    comm = XgmiAllReduce(1 << 20, device="cuda")
    params = [torch.nn.Parameter(_bf16((64,), 1))]
    opt = ShardedAdamW(comm, params, lr=1e-2)
    params[0].grad = torch.ones_like(params[0])
    opt.step(1)
    comm.close()
    return {"device": int(comm.device != DEV)}


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo", init_method=f"file://{os.environ['NETOP_INIT_FILE']}", rank=rank, world_size=world)
    torch.cuda.set_device(DEV)
    print("RESULT " + json.dumps(globals()["run_" + sys.argv[1]](rank, world, *sys.argv[2:])), flush=True)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()

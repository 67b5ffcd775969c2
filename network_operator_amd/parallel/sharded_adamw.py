"""AdamW with its states sharded over the ranks of a node, between the two phases of the direct
xGMI all-reduce.

The all-reduce of data-parallel gradients is a reduce-scatter and an all-gather
(:class:`~network_operator_amd.parallel.xgmi_comm.XgmiAllReduce`).  The optimizer's step fits
between them: rank d, which holds chunk d of the summed gradients anyway, updates chunk d of the
parameters with the states of that chunk alone, and the all-gather carries new parameters instead
of gradients -- the same bytes over the links, 1/n of the optimizer's memory and work on each GPU.

    comm = XgmiAllReduce(capacity_bytes=2 * sum(p.numel() + 8 for p in params) + 4096)
    opt = ShardedAdamW(comm, params, lr=3e-4, weight_decay=0.1, state_bits=8, max_norm=1.0)
    for step in range(1, steps + 1):
        loss(...).backward()
        norm = opt.step(step)

Reference counterpart: none (the reference has no GPU code).
"""

from __future__ import annotations

import math

from ..ops import adamw as A
from .xgmi_comm import XgmiAllReduce


class ShardedAdamW:
    """``params``: contiguous bf16 tensors on ``comm``'s device, the same on every rank (the
    constructor takes rank 0's layout for granted and every rank's values for equal).  Gradients are
    averaged over the ranks, in bf16 as they cross the links; masters and states are fp32, or 8-bit
    states (:class:`~network_operator_amd.ops.adamw.AdamW`, whose options these are), whose blocks start
    where a rank's part of a parameter does.  With ``max_norm`` gradients are clipped by the norm of all
    of them; a step whose norm is infinite or NaN changes nothing on any rank."""

    def __init__(self, comm: XgmiAllReduce, params, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 state_bits=32, seed=0, max_norm=None):
        import torch

        self.comm, self.params, self.max_norm = comm, list(params), max_norm
        if not self.params:
            raise ValueError("no parameters")
        for p in self.params:
            if p.dtype != torch.bfloat16 or not p.is_contiguous() or p.device != comm.device:
                raise ValueError("expected contiguous bfloat16 parameters on the communicator's device")
        A._refuse_shared(self.params)
        if max_norm is not None and not max_norm >= 0:
            raise ValueError("max_norm must not be negative")
        self.offsets, total = [], 0
        for p in self.params:
            self.offsets.append(total)
            total += -(-p.numel() // 8) * 8
        align = 8 * comm.world
        self.numel = max(-(-total // align) * align, align)
        self.chunk = self.numel // comm.world
        self.mine = slice(comm.rank * self.chunk, (comm.rank + 1) * self.chunk)
        comm.input(self.numel)  # capacity check
        flat = torch.zeros(self.numel, dtype=torch.bfloat16, device=comm.device)
        for p, at in zip(self.params, self.offsets):
            flat[at:at + p.numel()].copy_(p.detach().reshape(-1))
        self.shard = flat[self.mine].clone()
        # What lies here of each parameter is a tensor of the optimizer's: a block that shares a scale never
        # spans two.  Sizes of gap, part, gap, part ... for _parts; a rank of none has one empty part.
        self._sizes, end = [], 0
        for p, at in zip(self.params, self.offsets):
            a, b = (min(max(x - self.mine.start, 0), self.chunk) for x in (at, at + p.numel()))
            if a < b:
                self._sizes += [a - end, b - a]
                end = b
        self._sizes = self._sizes or [0, 0]
        self._sizes.append(self.chunk - end)
        # every rank its own random numbers: the chunks' positions all start at zero
        self.opt = A.AdamW(self._parts(self.shard), lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                           state_bits=state_bits, seed=(seed + 0x9E3779B1 * comm.rank) % (1 << 32))
        self._norm, self._coef = (torch.empty(1, device=comm.device) for _ in range(2))

    def _parts(self, chunk):
        """This rank's parts of the parameters, out of a chunk."""
        return list(chunk.split(self._sizes)[1::2])

    def state_dict(self) -> dict:
        """This rank's states (:meth:`AdamW.state_dict`); they belong to this rank, world size and order
        of parameters."""
        return self.opt.state_dict()

    def load_state_dict(self, state: dict) -> None:
        """Copies :meth:`state_dict`'s states in; the parameters, which the next step sets, are not touched."""
        self.opt.load_state_dict(state)
        for part, at in zip(self.opt.params, self.opt.offsets):
            part.copy_(self.opt.master[at:at + part.numel()])

    def _clip(self, grads) -> float:
        """``_coef`` for the norm over every rank's chunk, which it returns."""
        import torch.distributed as dist

        world = self.comm.world
        A.grad_norm([grads], self._norm, scale=1 / world)
        norms = [None] * world
        dist.all_gather_object(norms, float(self._norm), group=self.comm.group)
        total = math.sqrt(sum(x * x for x in norms))
        limit = math.inf if self.max_norm is None else self.max_norm
        self._coef.fill_(min(1.0, limit / (total + 1e-6)) / world if math.isfinite(total) else math.nan)
        return total

    def step(self, step: int, lr=None) -> float:
        """One step from the parameters' ``.grad`` (missing ones count as zeros); collective.
        ``step`` counts from 1.  Returns the gradients' norm before clipping."""
        import torch

        comm, n = self.comm, self.numel
        with torch.no_grad():
            x = comm.input(n)
            end = 0
            for p, at in zip(self.params, self.offsets):
                x[end:at].zero_()
                end = at + p.numel()
                if p.grad is None:
                    x[at:end].zero_()
                else:
                    x[at:end].copy_(p.grad.reshape(-1))
            x[end:].zero_()
            mine = comm.reduce_scatter(n)
            norm = self._clip(mine)
            self.opt.step(self._parts(mine), step=step, lr=lr, coef=self._coef)
            if not math.isfinite(norm):
                return norm  # the same on every rank: the parameters stay as they are
            mine.copy_(self.shard)
            full = comm.all_gather_inplace(n)
            for p, at in zip(self.params, self.offsets):
                p.copy_(full[at:at + p.numel()].view(p.shape))
        return norm

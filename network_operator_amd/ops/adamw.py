"""The optimizer's side of a data-parallel step: the global gradient norm and AdamW over many
tensors at once (``native/hip/adamw.hip``), for gradients that an all-reduce has summed (the hooks
of ``parallel/ddp_hooks.py``; ``parallel/sharded_adamw.py`` composes both with the reduce-scatter)::

    opt = AdamW(params, lr=3e-4, weight_decay=0.1, state_bits=8)
    total, coef = torch.empty(1, device=dev), torch.empty(1, device=dev)
    for step in range(1, steps + 1):
        ...                                             # backward, all-reduce
        grads = [p.grad for p in params]
        grad_norm(grads, total, coef=coef, max_norm=1.0)
        opt.step(grads, step=step, coef=coef)           # coef is read on the device

Both run on the tensors' device and its current stream, without a synchronisation, and can be
captured into a graph (``step`` and ``lr`` may be tensors there).  They raise if the library is
missing.
"""

from __future__ import annotations

import math
import struct
from array import array
from itertools import accumulate
from operator import attrgetter

from . import hip

BLOCK = 256  # elements of a tensor that share a scale; every tensor's states start at a whole block

# native/hip/adamw.hip:Hyper, StepParams and Held
_HELD = struct.Struct("=2Q2q")
_HYPER = struct.Struct("=9fI")
_STEP = struct.Struct("=8Q" + "9fI" + "6i")
_OVERLAP = -1


def _kinds():
    """Type codes, once torch is there (the package is imported without it too)."""
    global _KINDS
    import torch

    _KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    return _KINDS


_KINDS = None


_dtype, _shape = attrgetter("dtype"), attrgetter("shape")


def _gradients(grads):
    """The type and device that all ``grads`` but the ``None`` among them share, and their addresses."""
    import torch

    given = [g for g in grads if g is not None]
    if not given:
        return None, -1, [0] * len(grads)
    dtype, device = given[0].dtype, given[0].get_device()
    if dtype not in (_KINDS or _kinds()):
        raise ValueError(f"gradients: expected fp32, bf16 or fp16, got {dtype}")
    for other in set(map(_dtype, given)):
        if other is not dtype:
            raise ValueError(f"gradients must have one type: {dtype} and {other}")
    if not all(map(torch.Tensor.is_contiguous, given)):
        raise ValueError("gradients must be contiguous")
    if device < 0 or len(set(map(torch.Tensor.get_device, given))) > 1:
        raise ValueError("every tensor must be on one CUDA device")
    if len(given) == len(grads):
        return dtype, device, list(map(torch.Tensor.data_ptr, grads))
    return dtype, device, [0 if g is None else g.data_ptr() for g in grads]


def _refuse_shared(params):
    held = sorted((p.data_ptr(), p.numel() * p.element_size()) for p in params if p.numel())
    if any(a + n > b for (a, n), (b, _) in zip(held, held[1:])):
        raise ValueError("two parameters share memory")


def _one(t, dtype, device, what):
    if t.dtype != dtype or t.numel() != 1:
        raise ValueError(f"{what}: expected one {dtype} element")
    if t.get_device() != device:
        raise ValueError("every tensor must be on one CUDA device")
    return t.data_ptr()


def grad_norm(grads, total, *, norms=None, coef=None, max_norm=None, scale=1.0) -> None:
    """The 2-norm of all ``grads`` together, times ``scale`` (1 / ranks for summed gradients).

    ``grads``: contiguous tensors of one type (fp32, bf16 or fp16); ``None`` counts as zeros.
    ``total`` (fp32, one element) takes the norm; ``norms`` (fp32, one a gradient), where given, each
    gradient's own, times ``scale`` too; ``coef`` (fp32, one element), where given,
    ``scale * min(1, max_norm / (total + 1e-6))``, the factor :meth:`AdamW.step` takes (``scale``
    without ``max_norm``).  Where ``total`` is infinite (in fp32) or NaN ``coef`` is NaN, and that step is left out.

    Squares are summed in 64 bits, in an order that depends on the sizes alone: no square is too
    large or too small, and the same inputs give the same bits.
    """
    import torch

    limit = math.inf if max_norm is None else float(max_norm)
    if not limit >= 0:
        raise ValueError("max_norm must not be negative")
    if not 0 <= scale < math.inf:
        raise ValueError("scale must be finite and not negative")
    for t, what in ((total, "total"), (coef, "coef")):
        if t is not None and (t.dtype != torch.float32 or t.numel() != 1):
            raise ValueError(f"{what}: expected one {torch.float32} element")
    if norms is not None and (norms.dtype != torch.float32 or norms.shape != (len(grads),) or not norms.is_contiguous()):
        raise ValueError(f"norms: expected {len(grads)} contiguous float32 elements")
    dtype, device, ptrs = _gradients(grads)
    if dtype is None:
        raise ValueError("no gradients")
    for t in (total, coef, norms):
        if t is not None and t.get_device() != device:
            raise ValueError("every tensor must be on one CUDA device")
    ns = [0 if g is None else g.numel() for g in grads]
    elements = sum(ns)
    stretch = 1 << 13  # elements a workgroup: enough of them to fill the chip, few enough to add up
    while stretch < 1 << 16 and elements // stretch > 4096:
        stretch *= 2
    stretches = elements // stretch + len(ns)
    work = torch.empty(stretches + len(ns), dtype=torch.float64, device=total.device)
    table = array("Q", ptrs + ns)
    at = table.buffer_info()[0]
    rc = (hip._lib or hip.lib()).netop_grad_norm(
        at, at + 8 * len(ns), len(ns), _KINDS[dtype], stretch, work.data_ptr(), stretches, total.data_ptr(),
        0 if norms is None else norms.data_ptr(), 0 if coef is None else coef.data_ptr(), scale, limit, device,
        hip._raw_stream(device))
    if rc == _OVERLAP:
        raise ValueError("total, norms and coef must not share memory with each other or a gradient")
    hip._check(rc, "netop_grad_norm")
    hip._written([t for t in (total, norms, coef) if t is not None])


class AdamW:
    """AdamW over ``params`` (contiguous CUDA tensors of one type and device), with its states::

        g' = scale * coef * g
        m  = b1 m + (1 - b1) g'          v = b2 v + (1 - b2) g'^2
        p  = p (1 - lr wd) - lr (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps)

    fp32 parameters are updated in place.  bf16 and fp16 parameters are roundings of fp32 masters kept
    here (``master``, from the parameters' values at first): a step is mostly smaller than half a step
    of their own.

    ``state_bits=32`` keeps ``exp_avg`` (m) and ``exp_avg_sq`` (v) in fp32.  ``state_bits=8`` keeps
    m and sqrt(v) as e4m3 codes with one fp32 scale a block of 256 elements of a tensor
    (``exp_avg_scale``, ``exp_avg_sq_scale``; value = code * scale, v its square).  They are rounded
    up or down at random, in proportion, from a hash of (``seed``, ``step``, position): the same seed
    gives the same bits.  A sqrt(v) other than zero stays other than zero; a block whose m all lie
    below 2**-100 becomes zeros.

    All states are flat, with each tensor at a multiple of 256 elements (``offsets``); what lies
    between is zero.  The parameters must stay where they are: a step on one that has moved (``.data``
    replaced, ``module.to``) raises.  Steps on one object follow each other on one stream, or are
    ordered by the caller.
    """

    def __init__(self, params, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, seed=0):
        import torch

        kinds = _KINDS or _kinds()
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        first = self.params[0]
        self.dtype, self.device = first.dtype, first.device
        if self.dtype not in kinds:
            raise ValueError(f"parameters: expected fp32, bf16 or fp16, got {self.dtype}")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not all(0 <= b < 1 for b in betas) or len(betas) != 2:
            raise ValueError("betas must be two numbers in [0, 1)")
        if not 1e-30 <= eps < math.inf:  # zero would make 0 / 0 of an element that never had a gradient
            raise ValueError("eps must be positive")
        for name, x in (("lr", lr), ("weight_decay", weight_decay)):
            if not 0 <= x < math.inf:
                raise ValueError(f"{name} must not be negative")
        if not 0 <= seed < 1 << 32:
            raise ValueError("seed must fit 32 bits")
        for p in self.params:
            if p.dtype != self.dtype:
                raise ValueError(f"parameters must have one type: {self.dtype} and {p.dtype}")
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous")
        _refuse_shared(self.params)
        if not all(p.is_cuda and p.device == self.device for p in self.params):
            raise ValueError("every tensor must be on one CUDA device")
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), tuple(betas), float(eps), float(weight_decay)
        self.state_bits, self.seed = state_bits, seed
        self._kind, self._index = kinds[self.dtype], first.get_device()
        self._ptrs = [p.data_ptr() for p in self.params]
        self._shapes = [p.shape for p in self.params]
        ns = [p.numel() for p in self.params]
        self.offsets, total = [], 0
        for n in ns:
            self.offsets.append(total)
            total += -(-n // BLOCK) * BLOCK
        new = dict(device=self.device)
        codes = torch.float8_e4m3fn if state_bits == 8 else torch.float32
        self.exp_avg = torch.zeros(total, dtype=torch.uint8 if state_bits == 8 else codes, **new).view(codes)
        self.exp_avg_sq = torch.zeros_like(self.exp_avg.view(torch.uint8)).view(codes)
        self.exp_avg_scale = torch.zeros(total // BLOCK, **new) if state_bits == 8 else None
        self.exp_avg_sq_scale = torch.zeros(total // BLOCK, **new) if state_bits == 8 else None
        self.master = None
        if self._kind:
            self.master = torch.zeros(total, **new)
            for p, at, n in zip(self.params, self.offsets, ns):
                self.master[at:at + n].copy_(p.detach().reshape(-1))
        self._sizes = torch.tensor(ns, device="cpu")
        self._states = [t for t in (self.exp_avg, self.exp_avg_sq, self.master, self.exp_avg_scale, self.exp_avg_sq_scale)
                        if t is not None]
        self._all = [*self.params, *self._states]
        self._plan(ns)

    def _plan(self, ns):
        """The table of chunks, in launches of as many tensors as have room for their gradients' addresses."""
        import torch

        L = hip.lib()
        chunk, most = L.netop_adamw_chunk(), L.netop_adamw_max_grads()
        counts = [-(-n // chunk) for n in ns]
        # a row a tensor: its address, place in the states, elements, first chunk, chunks
        firsts = [0, *accumulate(counts)]
        rows = torch.tensor([self._ptrs, self.offsets, ns, firsts[:-1], counts], device=self.device)
        of = torch.repeat_interleave(torch.arange(len(ns), device=self.device), rows[4], output_size=firsts[-1])
        start = (torch.arange(firsts[-1], device=self.device) - rows[3][of]) * chunk
        self._table = torch.stack([rows[0][of] + start * self.params[0].element_size(), rows[1][of] + start, start,
                                   (rows[2][of] - start).clamp(max=chunk) | (of % most) << 32], 1)
        # What a step writes: address, end, and the parameter that it is.
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), i)
                       for i, t in [*enumerate(self.params), *((-1, t) for t in self._states)] if t.numel())
        self._spans, self._elements = array("q", [x for s in spans for x in s]), array("Q", ns)
        self._held = _HELD.pack(self._spans.buffer_info()[0], self._elements.buffer_info()[0], len(spans), len(ns))
        # (first tensor, one behind the last, address of its chunks, how many)
        at = self._table.data_ptr()
        self._launches = [(a, b, at + 32 * firsts[a], firsts[b] - firsts[a])
                          for a in range(0, len(ns), most) for b in (min(a + most, len(ns)),)]

    def state_dict(self) -> dict:
        """The states themselves (not copies), ``None`` for those this optimizer has not, and the tensors'
        ``sizes`` (int64, on the CPU)."""
        return dict(exp_avg=self.exp_avg, exp_avg_sq=self.exp_avg_sq, master=self.master,
                    exp_avg_scale=self.exp_avg_scale, exp_avg_sq_scale=self.exp_avg_sq_scale, sizes=self._sizes)

    def load_state_dict(self, state: dict) -> None:
        """Copies states in that :meth:`state_dict` of an optimizer over tensors of these sizes gave
        (where they have no ``sizes``, only the padded total is compared); the parameters are not touched."""
        mine = self.state_dict()
        sizes = mine.pop("sizes")
        if state.get("sizes") is not None and state["sizes"].tolist() != sizes.tolist():
            raise ValueError("states of tensors of other sizes")
        for k, t in mine.items():
            x = state.get(k)
            if (x is None) != (t is None) or t is not None and (x.shape != t.shape or x.dtype != t.dtype):
                raise ValueError(f"{k}: expected {None if t is None else (tuple(t.shape), t.dtype)}, "
                                 f"got {None if x is None else (tuple(x.shape), x.dtype)}")
        for k, t in mine.items():
            if t is not None:
                t.copy_(state[k])

    def step(self, grads, *, step, lr=None, coef=None, scale=1.0) -> None:
        """One step from ``grads``, one a parameter: contiguous, of its shape, all of one type (fp32,
        bf16 or fp16).  A parameter whose gradient is ``None`` is left as it is, with its states.  A
        gradient may be its own parameter's memory, element on element, but no other tensor's of this
        optimizer, and nor may ``coef``.

        ``step`` counts from 1: a number, or an int64 tensor of one element on the device (one below
        1 is taken for 1 there).  ``lr``
        replaces the constructor's: a number, or an fp32 tensor of one element.  ``coef`` (an fp32
        tensor of one element, from :func:`grad_norm`) and the number ``scale`` multiply the
        gradients; where the product with ``coef`` is not finite, nothing is changed.
        """
        import torch

        if len(grads) != len(self.params):
            raise ValueError(f"{len(self.params)} gradients expected, got {len(grads)}")
        if list(map(torch.Tensor.data_ptr, self.params)) != self._ptrs:
            raise ValueError("a parameter has moved since the optimizer was made")
        gtype, device, ptrs = _gradients(grads)
        if gtype is None:
            return
        if 0 in ptrs or list(map(_shape, grads)) != self._shapes:  # none given, or empty
            for g, shape in zip(grads, self._shapes):
                if g is not None and g.shape != shape:
                    raise ValueError(f"a gradient of shape {tuple(g.shape)} for a parameter of shape {tuple(shape)}")
        if device != self._index:
            raise ValueError("every tensor must be on one CUDA device")
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        coef_ptr = 0 if coef is None else _one(coef, torch.float32, device, "coef")
        (b1, b2), L, stream = self.betas, hip._lib or hip.lib(), hip._raw_stream(device)
        step_ptr = _one(step, torch.int64, device, "step") if isinstance(step, torch.Tensor) else 0
        lr_ptr = _one(lr, torch.float32, device, "lr") if isinstance(lr, torch.Tensor) else 0
        t = 1 if step_ptr else int(step)
        rate = self.lr if lr is None or lr_ptr else float(lr)
        if t < 1:
            raise ValueError("step counts from 1")
        if not 0 <= rate < math.inf:
            raise ValueError("lr must not be negative")
        key = (self.seed * 0x85EBCA6B + t * 0xC2B2AE35) & 0xFFFFFFFF
        hyper = (b1, 1 - b1, b2, 1 - b2, self.eps, 1 - rate * self.weight_decay, rate / (1 - b1 ** t),
                 1 / math.sqrt(1 - b2 ** t), scale, key ^ key >> 16)
        on_device = 0
        if step_ptr or lr_ptr:
            numbers = torch.empty(L.netop_adamw_hyper_bytes(), dtype=torch.uint8, device=self.device)
            on_device = numbers.data_ptr()
            hip._check(L.netop_adamw_hyper(on_device, _HYPER.pack(*hyper), b1, b2, rate, self.weight_decay, self.seed,
                                           lr_ptr, step_ptr, t, device, stream), "netop_adamw_hyper")
        eight = self.state_bits == 8
        table = array("Q", ptrs)
        at, held = table.buffer_info()[0], self._held
        for a, b, chunks, n in self._launches:
            if n == 0:
                continue  # nothing but empty tensors
            block = _STEP.pack(chunks, 0 if self.master is None else self.master.data_ptr(), self.exp_avg.data_ptr(),
                               self.exp_avg_sq.data_ptr(), self.exp_avg_scale.data_ptr() if eight else 0,
                               self.exp_avg_sq_scale.data_ptr() if eight else 0, coef_ptr, on_device, *hyper, n,
                               self._kind, _KINDS[gtype], self.state_bits, b - a, device)
            rc = L.netop_adamw_step(block, at, a, held, stream)
            if rc == _OVERLAP:
                raise ValueError("a gradient or coef lies in the memory of another tensor of this optimizer (a gradient "
                                 "may be its own parameter's memory, element on element)")
            hip._check(rc, "netop_adamw_step")
            held = None  # all of them have been looked up
        hip._written(self._all if 0 not in ptrs else
                     [*(p for p, g in zip(self.params, grads) if g is not None), *self._states])

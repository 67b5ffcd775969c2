"""The operators that follow a summed message, as cases to time: the residual RMS norm over
partial sums (tensor parallel), and the global gradient norm with the AdamW step over many tensors
(data parallel).  ``own = False`` computes each in elementary torch operations, ``own = True``
calls this package.

Layout of "many tensors": every tensor is a view of one flat buffer and starts at a multiple of
256 elements, the layout in which the optimizer keeps its own states; what lies between two
tensors is zero and stays zero.
"""

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # a block whose largest value is below is stored as zeros
BLOCK = 256  # elements of an optimizer state that share a scale
GROUP = 128  # columns of a norm's output that share a scale
EPS = 1e-6
BETA1, BETA2, ADAM_EPS, LR, DECAY = 0.9, 0.999, 1e-8, 3e-4, 0.1
SEED = 77  # of the 8-bit states' rounding


def listed():
    return [
        # One token of a served model between two layers: nothing but latency.
        dict(name="norm, one token", op="norm", rows=1, cols=4096, srcs=1, dtype="bf16", residual=True, out="same"),
        # A decode batch on 8 tensor-parallel ranks: each rank sums all eight partials itself.
        dict(name="norm, 64 tokens, 8 partials", op="norm", rows=64, cols=8192, srcs=8, dtype="bf16", residual=True,
             out="same"),
        # Prefill in front of an 8-bit product, a scale a row.
        dict(name="norm, prefill to e4m3 rows", op="norm", rows=16384, cols=8192, srcs=1, dtype="bf16", residual=True,
             out="e4m3_row"),
        # Odd width in half precision, a scale for each 128 columns, no residual stream yet (the first layer).
        dict(name="norm, odd fp16 to e4m3 groups", op="norm", rows=1001, cols=5003, srcs=3, dtype="fp16",
             residual=False, out="e4m3_128"),
        # A training step's backward pass through one norm, with the gradient of the residual stream.
        dict(name="norm backward, 8192 x 4096", op="norm_backward", rows=8192, cols=4096, dtype="bf16", residual=True),
        # The same where rows are few and wide and nothing is a multiple of eight.
        dict(name="norm backward, 333 x 10007", op="norm_backward", rows=333, cols=10007, dtype="fp32", residual=False),
        # The clip factor of one gradient bucket of a small model.
        dict(name="grad norm, 23 tensors", op="grad_norm", tensors=23, elements=1 << 20, dtype="fp32"),
        # ... and of 1 GiB of bf16 gradients, the fabric benchmark's message.
        dict(name="grad norm, 1 GiB bf16", op="grad_norm", tensors=290, elements=1 << 29, dtype="bf16"),
        # A small model's whole step: a call that is mostly launch and latency.
        dict(name="adamw, 23 tensors", op="adamw", tensors=23, elements=1 << 18, dtype="fp32", bits=32),
        # 1 GiB of bf16 gradients, fp32 masters and states.
        dict(name="adamw, 1 GiB bf16", op="adamw", tensors=290, elements=1 << 29, dtype="bf16", bits=32),
        # The same model's shard with 8-bit states.
        dict(name="adamw 8 bits, 0.5 GiB bf16", op="adamw", tensors=290, elements=1 << 28, dtype="bf16", bits=8),
        # Medium, odd, single precision throughout.
        dict(name="adamw 8 bits, 57 tensors", op="adamw", tensors=57, elements=(1 << 24) + 4711, dtype="fp32", bits=8),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_backward", "grad_norm", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("norm", "norm_backward"):
        cols = _spread(rng, 64, 20000)
        if rng.random() < 0.7:  # most widths are whole vectors
            cols = max(8, cols // 8 * 8)
        srcs = rng.choice([1, 1, 2, 3, 4, 8]) if op == "norm" else 1
        rows = _spread(rng, 1, max(2, (1 << 26) // cols // srcs))
        if op == "norm_backward":
            return dict(op=op, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.7)
        return dict(op=op, rows=rows, cols=cols, srcs=srcs, dtype=dtype, residual=rng.random() < 0.7,
                    out=rng.choice(["same", "same", "e4m3_row", "e4m3_128"]))
    elements = _spread(rng, 1 << 16, 1 << 27) + rng.randrange(100)
    tensors = _spread(rng, 1, 400)
    if op == "grad_norm":
        return dict(op=op, tensors=tensors, elements=elements, dtype=dtype)
    return dict(op=op, tensors=tensors, elements=elements, dtype=dtype, bits=rng.choice([8, 32]))


# ---- inputs -----------------------------------------------------------------------------------
def sizes(case):
    """The tensors' sizes: about half of them vectors (norm weights, biases), the others matrices of
    spread sizes that take up the rest; many are odd."""
    t, total = case["tensors"], case["elements"]
    rng = random.Random(t * 1000003 + total)
    small = [min(_spread(rng, 1, 8192), max(1, total // (2 * t))) for _ in range(t // 2)]
    share = [rng.uniform(0.2, 1.0) for _ in range(t - len(small))]
    left = total - sum(small)
    big = [max(1, int(left * s / sum(share))) for s in share]
    got = small + big
    rng.shuffle(got)
    return got


def _starts(ns):
    """Where each tensor starts in the flat buffer, and its length."""
    at, pos = [], 0
    for n in ns:
        at.append(pos)
        pos += (n + BLOCK - 1) // BLOCK * BLOCK
    return at, pos


def _mask(ns, at, flat):
    for n, a in zip(ns, at):
        flat[a + n:a + (n + BLOCK - 1) // BLOCK * BLOCK] = 0
    return flat


def _randn(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device=DEV, generator=gen) * scale).to(dtype)


def _quantised(x):
    """Blocks of an optimizer state as e4m3 codes and scales, rounded to nearest: a state to start from."""
    b = x.view(-1, BLOCK)
    amax = b.abs().amax(1)
    scale = torch.where(amax < TINY, 0, amax / E4M3_MAX)
    inv = torch.where(amax < TINY, 0, 1 / scale)
    return (b * inv[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).view(-1), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "norm":
        r, c, dt = case["rows"], case["cols"], TYPES[case["dtype"]]
        s["srcs"] = [_randn(gen, r, c, scale=0.5, dtype=dt) for _ in range(case["srcs"])]
        s["residual"] = _randn(gen, r, c, scale=2.0, dtype=dt) if case["residual"] else None
        s["weight"] = (1 + _randn(gen, c, scale=0.1)).to(dt)
        s["h"] = torch.empty(r, c, device=DEV, dtype=dt)
        s["rstd"] = torch.empty(r, device=DEV)
        s["out"] = torch.empty(r, c, device=DEV, dtype=dt if case["out"] == "same" else E4M3)
        groups = dict(same=None, e4m3_row=(r,), e4m3_128=(r, (c + GROUP - 1) // GROUP))[case["out"]]
        s["scales"] = torch.empty(groups, device=DEV) if groups else None
    elif case["op"] == "norm_backward":
        r, c, dt = case["rows"], case["cols"], TYPES[case["dtype"]]
        s["dy"] = _randn(gen, r, c, scale=0.1, dtype=dt)
        s["h"] = _randn(gen, r, c, scale=2.0, dtype=dt)
        s["dres"] = _randn(gen, r, c, scale=0.1, dtype=dt) if case["residual"] else None
        s["weight"] = (1 + _randn(gen, c, scale=0.1)).to(dt)
        s["rstd"] = torch.rsqrt(s["h"].float().square().mean(1) + EPS)
        s["dh"] = torch.empty(r, c, device=DEV, dtype=dt)
        s["dweight"] = torch.empty(c, device=DEV)
    else:
        dt = TYPES[case["dtype"]]
        ns = sizes(case)
        at, pos = _starts(ns)
        # fp16 gradients come with their loss scale: their squares would not be in range otherwise
        flat = _randn(gen, pos, scale=1.0 if case["dtype"] == "fp16" else 1e-3, dtype=dt)
        s["flat"] = _mask(ns, at, flat)
        s["grads"] = [flat[a:a + n] for a, n in zip(at, ns)]
        if case["op"] == "grad_norm":
            s["norms"] = torch.empty(len(ns), device=DEV)
            s["total"], s["coef"] = torch.empty(1, device=DEV), torch.empty(1, device=DEV)
            return s
        s["coef"] = torch.full((1,), 0.7e-3 if case["dtype"] == "fp16" else 0.7, device=DEV)
        p = _mask(ns, at, _randn(gen, pos, scale=0.02))
        m = _mask(ns, at, _randn(gen, pos, scale=3e-4))
        v = _mask(ns, at, _randn(gen, pos, scale=6e-4)).square_()
        s["step"] = 100
        s["p"] = p if dt == torch.float32 else p.to(dt)
        if dt != torch.float32:
            s["master"] = p
        if case["bits"] == 8:
            s["m"], s["m_scale"] = _quantised(m)
            s["v"], s["v_scale"] = _quantised(v.sqrt_())
        else:
            s["m"], s["v"] = m, v
        if own:
            from network_operator_amd.ops import adamw

            opt = adamw.AdamW([s["p"][a:a + n] for a, n in zip(at, ns)], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                              weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
            opt.load_state_dict(dict(exp_avg=s["m"], exp_avg_sq=s["v"], master=s.get("master"),
                                     exp_avg_scale=s.get("m_scale"), exp_avg_sq_scale=s.get("v_scale")))
            s["opt"] = opt
            for k in ("m", "v", "master", "m_scale", "v_scale"):
                s.pop(k, None)
    return s


# ---- one pass ---------------------------------------------------------------------------------
def run(s):
    return dict(norm=_norm, norm_backward=_norm_backward, grad_norm=_grad_norm, adamw=_adamw)[s["case"]["op"]](s)


def _norm(s):
    if own:
        from network_operator_amd.ops import norm

        norm.add_rms_norm(s["srcs"], s["weight"], s["out"], residual=s["residual"], residual_out=s["h"],
                          rstd=s["rstd"], scales=s["scales"], eps=EPS)
        return {k: s[k] for k in ("out", "h", "rstd", "scales")}
    dt = s["srcs"][0].dtype
    h = torch.stack(s["srcs"]).float().sum(0) if len(s["srcs"]) > 1 else s["srcs"][0].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    rstd = 1 / torch.sqrt((h * h).mean(1) + EPS)
    y = h * rstd[:, None] * s["weight"].float()
    if s["scales"] is None:
        return dict(out=y.to(dt), h=h.to(dt), rstd=rstd, scales=None)
    r, c = y.shape
    g = c if s["scales"].dim() == 1 else GROUP
    y = torch.nn.functional.pad(y, (0, -c % g)).view(r, -1, g)
    amax = y.abs().amax(2)
    scale = torch.where(amax < TINY, 0, amax / E4M3_MAX)
    q = (y * torch.where(amax < TINY, 0, 1 / scale)[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(r, -1)[:, :c].to(E4M3)
    return dict(out=q, h=h.to(dt), rstd=rstd, scales=scale.view(s["scales"].shape))


def _norm_backward(s):
    if own:
        from network_operator_amd.ops import norm

        norm.add_rms_norm_backward(s["dy"], s["h"], s["weight"], s["rstd"], s["dh"], s["dweight"], dresidual=s["dres"])
        return dict(dh=s["dh"], dweight=s["dweight"])
    dy, h, r = s["dy"].float(), s["h"].float(), s["rstd"][:, None]
    a = dy * s["weight"].float()
    dh = r * a - h * (r * r * r * (a * h).mean(1, keepdim=True))
    if s["dres"] is not None:
        dh = dh + s["dres"].float()
    return dict(dh=dh.to(s["dy"].dtype), dweight=(dy * h * r).sum(0))


def _grad_norm(s):
    if own:
        from network_operator_amd.ops import adamw

        adamw.grad_norm(s["grads"], s["total"], norms=s["norms"], coef=s["coef"], max_norm=1.0, scale=0.125)
        return {k: s[k] for k in ("total", "coef", "norms")}
    sums = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    total = 0.125 * sums.sum().sqrt()
    coef = 0.125 * torch.clamp(1.0 / (total + 1e-6), max=1.0)
    return dict(total=total.float().view(1), coef=coef.float().view(1), norms=(0.125 * sums.sqrt()).float())


def _random16(n, step):
    """Two 16-bit random numbers for each position of the flat buffer: a hash of (seed, step, position)."""
    full = 0xFFFFFFFF
    key = (SEED * 0x85EBCA6B + step * 0xC2B2AE35) & full
    key ^= key >> 16
    i = torch.arange(n, device=DEV)
    x = ((i & full) * 0x9E3779B1 & full) ^ ((i >> 32) * 0x85EBCA77 & full) ^ key
    x = ((x ^ (x >> 15)) * 0x2C1B3C6D) & full
    x = ((x ^ (x >> 12)) * 0x297A2D39) & full
    x = x ^ (x >> 15)
    return x & 0xFFFF, x >> 16


def _stochastic(x, rnd, keep):
    """Blocks of x as e4m3 codes and scales: a value between two codes becomes the upper one where
    its place between them plus the random number / 2^16 reaches one.  ``keep``: a value other than
    zero does not become zero."""
    b = x.view(-1, BLOCK)
    amax = b.abs().amax(1)
    scale = torch.where(amax < TINY, 0, amax / E4M3_MAX)
    u = (b.abs() * torch.where(amax < TINY, 0, 1 / scale)[:, None]).clamp(max=E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(u)).clamp(min=-6) - 3)
    # log2 rounds: just below a power of two it may already give that power
    step = torch.where((u < 8 * step) & (step > 2.0 ** -9), step / 2, step)
    k = torch.floor(u / step + rnd.view(-1, BLOCK).float() / 65536)
    if keep:
        k = torch.where((k == 0) & (u > 0), 1, k)
    return (k * step * b.sign()).to(E4M3).view(-1), scale


def _adamw(s):
    s["step"] += 1
    if own:
        s["opt"].step(s["grads"], step=s["step"], coef=s["coef"])
        d = s["opt"].state_dict()
        return dict(p=s["p"], master=d["master"], m=d["exp_avg"], v=d["exp_avg_sq"], m_scale=d["exp_avg_scale"],
                    v_scale=d["exp_avg_sq_scale"])
    eight = s["case"]["bits"] == 8
    m, v = s["m"], s["v"]
    if eight:
        m = (m.view(-1, BLOCK).float() * s["m_scale"][:, None]).view(-1)
        v = (v.view(-1, BLOCK).float() * s["v_scale"][:, None]).view(-1).square()
    g = s["flat"].float() * s["coef"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    c1, c2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    w = s["master"] if "master" in s else s["p"]
    w.copy_(w * (1 - LR * DECAY) - LR * (m / c1) / (torch.sqrt(v / c2) + ADAM_EPS))
    if "master" in s:
        s["p"].copy_(w)
    if eight:
        rm, rv = _random16(m.numel(), s["step"])
        s["m"], s["m_scale"] = _stochastic(m, rm, False)
        s["v"], s["v_scale"] = _stochastic(torch.sqrt(v), rv, True)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return {k: s.get(k) for k in ("p", "master", "m", "v", "m_scale", "v_scale")}


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    width = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        eight = case["out"] != "same"
        scales = 0 if not eight else case["rows"] * (1 if case["out"] == "e4m3_row" else -(-case["cols"] // GROUP))
        moved = n * (width * (case["srcs"] + case["residual"] + 1) + (1 if eight else width))
        return dict(bytes=moved + case["cols"] * width + case["rows"] * 4 + scales * 4, flops=n * (case["srcs"] + 6))
    if case["op"] == "norm_backward":
        n = case["rows"] * case["cols"]
        return dict(bytes=n * width * (3 + case["residual"]) + case["cols"] * (width + 4) + case["rows"] * 4,
                    flops=n * 12)
    n = sum(sizes(case))
    if case["op"] == "grad_norm":
        return dict(bytes=n * width + case["tensors"] * 4 + 8, flops=2 * n)
    per = width + (8 if width == 4 else 10) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    return dict(bytes=n * per, flops=n * 18)


# ---- the same from the definitions in 64 bits -------------------------------------------------
def _e4m3_codes():
    """The values of e4m3 from zero up: exponent and fraction fields read out of each code."""
    got = [(c & 7) / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)]
    return torch.tensor(got, dtype=torch.float64, device=DEV)


def _nearest_code(u):
    codes = _e4m3_codes()
    a = u.abs().clamp(max=E4M3_MAX).contiguous()
    hi = torch.searchsorted(codes, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = codes[hi] - a, a - codes[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(codes[pick], u)


def _exact_norm(s, case):
    h = s["residual"].double() if s["residual"] is not None else torch.zeros_like(s["h"], dtype=torch.float64)
    for x in s["srcs"]:
        h += x.double()
    rstd = (torch.linalg.vector_norm(h, dim=1).square() / case["cols"] + EPS).pow(-0.5)
    y = torch.einsum("rc,r,c->rc", h, rstd, s["weight"].double())
    if case["out"] == "same":
        return dict(out=y, h=h, rstd=rstd, scales=None)
    width = case["cols"] if case["out"] == "e4m3_row" else GROUP
    parts = y.split(width, dim=1)
    scales = torch.stack([p.abs().max(1).values / E4M3_MAX for p in parts], 1)
    out = torch.cat([_nearest_code(p / scales[:, i:i + 1]) for i, p in enumerate(parts)], 1)
    return dict(out=out, h=h, rstd=rstd, scales=scales.reshape(s["scales"].shape))


def _exact_norm_backward(s, case):
    dy, h, r, w = (s[k].double() for k in ("dy", "h", "rstd", "weight"))
    xhat = h * r[:, None]
    dxhat = dy * w
    dh = (dxhat - xhat * (dxhat * xhat).sum(1, keepdim=True) / case["cols"]) * r[:, None]
    if s["dres"] is not None:
        dh += s["dres"].double()
    return dict(dh=dh, dweight=(dy * xhat).sum(0))


def _exact_grad_norm(s):
    norms = torch.stack([torch.linalg.vector_norm(g, dtype=torch.float64) for g in s["grads"]]) / 8
    total = torch.linalg.vector_norm(norms)
    factor = min(1.0, 1.0 / (float(total) + 1e-6)) / 8
    return dict(total=total.view(1), coef=torch.full((1,), factor, dtype=torch.float64), norms=norms)


def _exact_states(x, rnd, keep):
    """x (blocks of a state) as codes' values and scales; ``rnd`` in [0, 1)."""
    amax = x.abs().max(1, keepdim=True).values
    scale = amax / E4M3_MAX
    u = torch.where(amax > 0, x.abs() / scale, 0).clamp(max=E4M3_MAX)
    codes = _e4m3_codes()
    lo = (torch.searchsorted(codes, u, right=True) - 1).clamp(max=125)
    place = (u - codes[lo]) / (codes[lo + 1] - codes[lo])
    pick = torch.where(place + rnd >= 1, lo + 1, lo)
    if keep:
        pick = torch.where(u > 0, pick.clamp(min=1), pick)
    return torch.copysign(codes[pick], x), scale[:, 0]


def _exact_adamw(s, case):
    t = s["step"] + 1
    eight = case["bits"] == 8
    w0 = s.get("master", s["p"])
    kept = dict(p=[], m=[], v=[], m_scale=[], v_scale=[])
    span = 1 << 24  # a stretch of the flat buffer at a time: 64-bit copies of all of it would not fit
    for a in range(0, w0.numel(), span):
        b = min(a + span, w0.numel())
        at = slice(a, b)
        g = s["flat"][at].double() * s["coef"].double()
        m, v = s["m"][at].to(torch.float64), s["v"][at].to(torch.float64)
        if eight:
            blocks = slice(a // BLOCK, b // BLOCK)
            m = m * s["m_scale"][blocks].double().repeat_interleave(BLOCK)
            v = (v * s["v_scale"][blocks].double().repeat_interleave(BLOCK)) ** 2
        m = torch.lerp(g, m, BETA1)
        v = torch.lerp(g ** 2, v, BETA2)
        w = w0[at].double()
        w = w - LR * DECAY * w - LR * (m / -math.expm1(t * math.log(BETA1))) / (
            (v / -math.expm1(t * math.log(BETA2))).sqrt() + ADAM_EPS)
        kept["p"].append(w)
        if not eight:
            kept["m"].append(m)
            kept["v"].append(v)
            continue
        x = torch.arange(a, b, device=DEV)  # positions here stay below 2^32
        x = (x * 0x9E3779B1) % (1 << 32)
        key = (SEED * 0x85EBCA6B + t * 0xC2B2AE35) % (1 << 32)
        x ^= key ^ (key >> 16)
        x ^= x >> 15
        x = (x * 0x2C1B3C6D) % (1 << 32)
        x ^= x >> 12
        x = (x * 0x297A2D39) % (1 << 32)
        x ^= x >> 15
        for name, y, r in (("m", m, x % 65536), ("v", v.sqrt(), x // 65536)):
            q, scale = _exact_states(y.view(-1, BLOCK), r.view(-1, BLOCK).double() / 65536, name == "v")
            kept[name].append(q.view(-1))
            kept[name + "_scale"].append(scale)
    got = {k: torch.cat(x) if x else None for k, x in kept.items()}
    got["master"] = got["p"] if "master" in s else None
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s, case)
    if case["op"] == "norm_backward":
        return _exact_norm_backward(s, case)
    return _exact_grad_norm(s) if case["op"] == "grad_norm" else _exact_adamw(s, case)

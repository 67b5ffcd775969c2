"""The gradient norm and the AdamW step over many tensors (ops/adamw.py) against their definitions
in 64 bits.  Tolerances count roundings: half a step of a stored type, 2^-24 of the magnitudes that
go into each fp32 operation."""

import math

import pytest

torch = pytest.importorskip("torch")

from network_operator_amd.ops import adamw  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3 = torch.float8_e4m3fn
ULP = 2.0 ** -24
SIZES = [1, 3, 255, 256, 257, 0, 4095, 4096, 4097, 70001, 12, 9000]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _tensors(sizes, dtype, dev, scale, seed, odd=False):
    """Views of one buffer, at odd offsets if asked, and that buffer."""
    gap = 3 if odd else 0
    g = torch.Generator().manual_seed(seed)
    buf = (torch.randn(sum(sizes) + gap * (len(sizes) + 1), generator=g) * scale).to(dtype).to(dev)
    got, at = [], gap
    for n in sizes:
        got.append(buf[at:at + n])
        at += n + gap
    return got, buf


def _codes():
    return torch.arange(127, dtype=torch.uint8).view(E4M3).double()


def _hash(i, seed, step):
    full = 0xFFFFFFFF
    key = (seed * 0x85EBCA6B + step * 0xC2B2AE35) & full
    x = ((i & full) * 0x9E3779B1 & full) ^ ((i >> 32) * 0x85EBCA77 & full) ^ key ^ (key >> 16)
    x = (x ^ x >> 15) * 0x2C1B3C6D & full
    x = (x ^ x >> 12) * 0x297A2D39 & full
    x = x ^ x >> 15
    return (x & 0xFFFF).double() / 65536, (x >> 16).double() / 65536


def _moments(opt, i):
    """m and v of tensor i as the optimizer keeps them, in 64 bits on the CPU."""
    at, n = opt.offsets[i], opt.params[i].numel()
    pad = slice(at, at + -(-n // 256) * 256)
    m, v = (t[pad].cpu().double() if opt.state_bits == 32 else t[pad].cpu().float().double()
            for t in (opt.exp_avg, opt.exp_avg_sq))
    if opt.state_bits == 8:
        b = slice(at // 256, at // 256 + -(-n // 256))
        m = m * opt.exp_avg_scale[b].cpu().double().repeat_interleave(256)
        v = (v * opt.exp_avg_sq_scale[b].cpu().double().repeat_interleave(256)) ** 2
    return m[:n], v[:n]


def _expected(p, g, m, v, step, lr, betas, eps, weight_decay):
    """The new p, m and v, the magnitudes that went into m, and how far p moves for such an m."""
    b1, b2 = betas
    mag = abs(b1 * m) + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    rate = lr / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p * (1 - lr * weight_decay) - rate * m, m, v, mag, rate * mag


def _close(got, want, tol):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than allowed, {int((off > tol).sum())} values"


def _check_codes(x, mag, got, scale, rnd, keep):
    """got (codes' values) of one tensor against x in 64 bits, to which magnitudes `mag` were added up."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    amax = blocks.abs().amax(1)
    most = torch.nn.functional.pad(mag, (0, -n % 256)).view(-1, 256).amax(1)
    _close(scale, torch.where(amax < 2.0 ** -100, 0, amax / 448), 8 * ULP * most / 448)
    per = scale.cpu().double().repeat_interleave(256)[:n]
    u = torch.where(per > 0, x.abs() / per.clamp(min=1e-300), 0).clamp(max=448)
    codes = _codes()
    lo = (torch.searchsorted(codes, u, right=True) - 1).clamp(max=125)
    place = (u - codes[lo]) / (codes[lo + 1] - codes[lo])
    up = place + rnd >= 1
    # fp32 may decide a value at the border otherwise: 8 roundings of what was added up, in codes' distances
    edge = 1e-4 + 16 * 8 * ULP * mag / x.abs().clamp(min=1e-300)
    sure = ((place + rnd - 1).abs() > edge) & (place > edge) & (place < 1 - edge)
    want = torch.where(up, codes[lo + 1], codes[lo])
    want = torch.where((want == 0) & (u > 0), codes[1], want) if keep else want
    got = got.cpu().float().double()
    assert bool((got.abs()[sure] == want[sure]).all())
    step = codes[lo + 1] - codes[lo]
    assert bool(((got.abs() - u).abs() <= step * 1.01).all())
    assert bool((got * x >= 0).all())
    if keep:
        assert bool(((got > 0) == (u > 0)).all())
    assert int(sure.sum()) > 0.9 * n or n < 300


def _run_and_check(dev, sizes, ptype, gtype, bits, steps=3, odd=False, coef=0.5, scale=0.25, seed=5):
    params, buf = _tensors(sizes, ptype, dev, 0.5, 1, odd)
    before = buf.clone()
    opt = adamw.AdamW(params, state_bits=bits, seed=seed, **HYPER)
    c = torch.full((1,), coef, device=dev)
    for step in range(1, steps + 1):
        grads, _ = _tensors(sizes, gtype, dev, 0.1, 10 + step, odd)
        old = [(p.detach().double().cpu() if opt.master is None else
                opt.master[a:a + p.numel()].double().cpu(), *_moments(opt, i))
               for i, (p, a) in enumerate(zip(params, opt.offsets))]
        opt.step(grads, step=step, coef=c, scale=scale)
        for i, (p, at) in enumerate(zip(params, opt.offsets)):
            n = p.numel()
            if not n:
                continue
            g = grads[i].double().cpu() * (coef * scale)
            w, m, v, mag, u = _expected(*(old[i][0], g, *old[i][1:]), step, **HYPER)
            w_tol = ULP * (4 * w.abs() + 4 * old[i][0].abs() + 16 * u.abs()) + 1e-12
            if opt.master is None:
                _close(p, w, w_tol)
            else:
                master = opt.master[at:at + n]
                _close(master, w, w_tol)
                assert torch.equal(p, master.to(ptype))
            if bits == 32:
                _close(opt.exp_avg[at:at + n], m, ULP * 4 * (old[i][1].abs() + g.abs()))
                _close(opt.exp_avg_sq[at:at + n], v, ULP * 6 * v)
            else:
                rm, rv = _hash(torch.arange(at, at + n), seed, step)
                b = slice(at // 256, at // 256 + -(-n // 256))
                _check_codes(m, mag, opt.exp_avg[at:at + n], opt.exp_avg_scale[b], rm, False)
                _check_codes(v.sqrt(), v.sqrt(), opt.exp_avg_sq[at:at + n], opt.exp_avg_sq_scale[b], rv, True)
    kept = torch.ones(buf.numel(), dtype=torch.bool, device=dev)  # what lies between the tensors
    for p in params:
        a = (p.data_ptr() - buf.data_ptr()) // p.element_size() if p.numel() else 0
        kept[a:a + p.numel()] = False
    assert torch.equal(buf[kept], before[kept])
    used = torch.zeros(opt.exp_avg.numel(), dtype=torch.bool)
    for p, a in zip(params, opt.offsets):
        used[a:a + p.numel()] = True
    for t in (opt.exp_avg, opt.exp_avg_sq, opt.master):
        assert t is None or bool((t.float().cpu()[~used] == 0).all())
    return opt


# ---- refusals (no GPU) ------------------------------------------------------------------------
@pytest.mark.parametrize("params,kw,why", [
    ([], {}, "no parameters"),
    ([torch.zeros(8, dtype=torch.float64)], {}, "expected fp32, bf16 or fp16"),
    ([torch.zeros(8), torch.zeros(8, dtype=BF16)], {}, "one type"),
    ([torch.zeros(8, 8).t()], {}, "contiguous"),
    ([torch.zeros(8)], dict(state_bits=16), "8 or 32"),
    ([torch.zeros(8)], dict(betas=(0.9, 1.0)), "betas"),
    ([torch.zeros(8)], dict(betas=(0.9,)), "betas"),
    ([torch.zeros(8)], dict(eps=0.0), "eps"),
    ([torch.zeros(8)], dict(lr=-1.0), "lr"),
    ([torch.zeros(8)], dict(lr=float("nan")), "lr"),
    ([torch.zeros(8)], dict(weight_decay=-0.1), "weight_decay"),
    ([torch.zeros(8)], dict(seed=1 << 32), "seed"),
    ([torch.zeros(16)[:9], torch.zeros(1)], {}, "one CUDA device"),
])
def test_adamw_refuses(params, kw, why):
    with pytest.raises(ValueError, match=why):
        adamw.AdamW(params, **{"lr": 1e-3, **kw})


def test_adamw_refuses_shared_memory():
    b = torch.zeros(16)
    for pair in ([b, b], [b[:9], b[8:]], [b, b[3:4]]):
        with pytest.raises(ValueError, match="share memory"):
            adamw.AdamW(pair, lr=1e-3)


@pytest.mark.parametrize("grads,kw,why", [
    ([], {}, "no gradients"),
    ([None, None], {}, "no gradients"),
    ([torch.zeros(8, dtype=torch.float64)], {}, "expected fp32, bf16 or fp16"),
    ([torch.zeros(8), torch.zeros(8, dtype=BF16)], {}, "one type"),
    ([torch.zeros(8, 8).t()], {}, "contiguous"),
    ([torch.zeros(8)], dict(max_norm=-1.0), "max_norm"),
    ([torch.zeros(8)], dict(max_norm=float("nan")), "max_norm"),
    ([torch.zeros(8)], dict(scale=float("inf")), "scale"),
    ([torch.zeros(8)], dict(total=torch.zeros(2)), "total: expected one"),
    ([torch.zeros(8)], dict(coef=torch.zeros(1, dtype=torch.float64)), "coef: expected one"),
    ([torch.zeros(8)], dict(norms=torch.zeros(2)), "norms: expected 1"),
    ([torch.zeros(8)], {}, "one CUDA device"),
])
def test_grad_norm_refuses(grads, kw, why):
    kw = dict(kw)
    total = kw.pop("total", torch.zeros(1))
    with pytest.raises(ValueError, match=why):
        adamw.grad_norm(grads, total, **kw)


@pytest.mark.gpu
def test_step_refuses(cuda_device):
    p = [torch.zeros(8, 4, device=cuda_device), torch.zeros(5, device=cuda_device)]
    opt = adamw.AdamW(p, lr=1e-3)
    g = [torch.zeros_like(x) for x in p]
    one = torch.ones(1, device=cuda_device)
    for grads, kw, why in [(g[:1], {}, "2 gradients expected"), ([g[0], g[1].to(BF16)], {}, "one type"),
                           ([g[0].view(4, 8), g[1]], {}, "of shape"), ([torch.zeros(4, 8, device=cuda_device).t(), g[1]], {}, "contiguous"),
                           ([g[0].cpu(), g[1]], {}, "one CUDA device"), ([x.double() for x in g], {}, "expected fp32"),
                           (g, dict(step=0), "counts from 1"), (g, dict(step=one), "step: expected one"), (g, dict(lr=-1.0), "lr"),
                           (g, dict(coef=one.cpu()), "one CUDA device"), (g, dict(coef=one.double()), "coef: expected"),
                           (g, dict(scale=float("nan")), "scale")]:
        with pytest.raises(ValueError, match=why):
            opt.step(grads, **{"step": 1, **kw})
    with pytest.raises(ValueError, match="exp_avg_scale"):
        opt.load_state_dict({**opt.state_dict(), "exp_avg_scale": one})
    assert all(bool((x == 0).all()) for x in p)
    p[1].data = torch.zeros(5, device=cuda_device)
    with pytest.raises(ValueError, match="has moved"):
        opt.step(g, step=1)


# ---- AdamW ------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gtype", [F32, BF16, F16])
@pytest.mark.parametrize("ptype", [F32, BF16, F16])
def test_steps(cuda_device, ptype, gtype, bits):
    _run_and_check(cuda_device, SIZES, ptype, gtype, bits)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_views_at_odd_offsets(cuda_device, bits):
    _run_and_check(cuda_device, SIZES, BF16, BF16, bits, odd=True)
    _run_and_check(cuda_device, SIZES[:6], F32, F16, bits, odd=True)


@pytest.mark.gpu
def test_more_tensors_than_one_launch_takes(cuda_device):
    opt = _run_and_check(cuda_device, [(7 * i) % 600 for i in range(1000)], BF16, F32, 8, steps=1)
    assert len(opt._launches) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_steps_of_torch(cuda_device, bits):
    """Twenty steps of the same gradients as torch.optim.AdamW in 64 bits.  With 32 bits each step
    adds some roundings.  With 8, m carries a noise of a tenth (3.7 % a rounding, for some ten steps)
    and sqrt(v) one of a third (it moves by ever less than a code's distance of 9 %, up or down by all
    of it): what the parameters have gone is off by less than 0.45 of its length, a cosine of 0.9."""
    p0 = torch.randn(5000, device=cuda_device)
    mine, ref = p0.clone(), torch.nn.Parameter(p0.double())
    opt, other = adamw.AdamW([mine], state_bits=bits, **HYPER), torch.optim.AdamW([ref], **HYPER, foreach=False)
    mean = torch.randn(5000, device=cuda_device)
    for step in range(1, 21):
        g = mean + torch.randn(5000, device=cuda_device)
        ref.grad = g.double()
        other.step()
        opt.step([g], step=step)
    gone, want = mine.double() - p0.double(), ref.detach() - p0.double()
    if bits == 32:
        assert float((mine.double() - ref.detach()).abs().max()) <= 20 * ULP * (8 * float(p0.abs().max()) + 16 * 0.003)
    else:
        assert float((gone * want).sum() / gone.norm() / want.norm()) > 0.9


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_no_gradient_and_overflowed_gradients_change_nothing(cuda_device, bits):
    params, buf = _tensors([300, 5, 4100], BF16, cuda_device, 1.0, 2)
    grads, _ = _tensors([300, 5, 4100], BF16, cuda_device, 1.0, 3)
    opt = adamw.AdamW(params, state_bits=bits, **HYPER)
    opt.step(grads, step=1)
    keep = [t.clone() for t in (buf, *(x for x in opt.state_dict().values() if x is not None))]

    def changed():
        now = (buf, *(x for x in opt.state_dict().values() if x is not None))
        return not all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(keep, now))

    for bad in (float("nan"), float("inf")):
        opt.step(grads, step=2, coef=torch.full((1,), bad, device=cuda_device))
    opt.step([None] * 3, step=2)
    assert not changed()
    kept = params[1].clone()
    opt.step([grads[0], None, grads[2]], step=2)
    assert torch.equal(params[1], kept) and changed()
    assert torch.equal(opt.exp_avg[opt.offsets[1]:opt.offsets[1] + 256].view(torch.uint8),
                       keep[1][opt.offsets[1]:opt.offsets[1] + 256].view(torch.uint8))


@pytest.mark.gpu
def test_a_non_finite_gradient_stays_in_its_element_or_block(cuda_device):
    for bits in (32, 8):
        p = torch.zeros(1024, device=cuda_device)
        opt = adamw.AdamW([p], state_bits=bits, **HYPER)
        g = torch.ones(1024, device=cuda_device)
        g[300] = float("nan")
        opt.step([g], step=1)
        at = torch.arange(1024, device=cuda_device) == 300
        assert bool(torch.isnan(p[at]).all()) and bool(torch.isfinite(p[~at]).all())
        assert bool(torch.isnan(opt.exp_avg.float()[at]).all()) and bool(torch.isfinite(opt.exp_avg.float()[~at]).all())
        g[300], g[700] = 1, float("inf")
        opt.step([g], step=2)
        other = torch.arange(1024, device=cuda_device) // 256 != 2
        assert bool(torch.isfinite(p[other & ~at]).all())


@pytest.mark.gpu
def test_one_seed_gives_the_same_bits_and_another_gives_others(cuda_device):
    got = []
    for seed in (1, 1, 2):
        params, _ = _tensors([5000, 77], F32, cuda_device, 1.0, 4)
        opt = adamw.AdamW(params, state_bits=8, seed=seed, **HYPER)
        for step in (1, 2):
            opt.step(_tensors([5000, 77], F32, cuda_device, 1.0, 5 + step)[0], step=step)
        got.append(torch.cat([opt.exp_avg.view(torch.uint8), opt.exp_avg_sq.view(torch.uint8)]))
    assert torch.equal(got[0], got[1]) and not torch.equal(got[0], got[2])


@pytest.mark.gpu
def test_eight_bit_second_moments_move_by_less_than_a_code(cuda_device):
    """With b2 = 0.999 and no gradient but in one element a block, the others' v fall by 0.999 a step,
    far less than half a code: on average they have to follow all the same.  After 400 steps a value
    is exp(-0.4) of the first; each value has a random walk of its own, the mean over 2^18 does not."""
    n = 1 << 18
    p = torch.zeros(n, device=cuda_device)
    opt = adamw.AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    g = torch.rand(n, device=cuda_device) + 0.5
    g[::256] = 4.0
    for step in range(1, 20):
        opt.step([g], step=step)
    idle = torch.arange(n, device=cuda_device) % 256 != 0
    root = lambda: (opt.exp_avg_sq.float().view(-1, 256) * opt.exp_avg_sq_scale[:, None]).view(-1)[idle].double()  # noqa: E731
    first = root().mean()
    g[idle] = 0
    for step in range(20, 420):
        opt.step([g], step=step)
    # a rounding's mean is exact to 2^-17 of a code's distance (1/8 of a value): 400 of them 4e-4;
    # the elements' own walks, four tenths each, 0.4 / 2^9 = 8e-4
    assert abs(float(root().mean() / first) - 0.999 ** 200) < 5e-3


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_states_are_saved_and_loaded(cuda_device, bits):
    def fresh():
        params, _ = _tensors([700, 33], F16, cuda_device, 1.0, 6)
        return params, adamw.AdamW(params, state_bits=bits, **HYPER)

    (pa, a), (pb, b) = fresh(), fresh()
    for step in (1, 2):
        a.step(_tensors([700, 33], BF16, cuda_device, 1.0, step)[0], step=step)
    b.load_state_dict(a.state_dict())
    a.step(_tensors([700, 33], BF16, cuda_device, 1.0, 3)[0], step=3)
    b.step(_tensors([700, 33], BF16, cuda_device, 1.0, 3)[0], step=3)
    assert all(torch.equal(x, y) for x, y in zip(pa, pb))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_with_step_and_lr_on_the_device(cuda_device, bits):
    """Norm and step captured; each replay, with eager work between, against the same eager step."""
    sizes = [5000, 1, 300]
    (pa, _), (pb, _) = _tensors(sizes, BF16, cuda_device, 1.0, 7), _tensors(sizes, BF16, cuda_device, 1.0, 7)
    a, b = adamw.AdamW(pa, state_bits=bits, **HYPER), adamw.AdamW(pb, state_bits=bits, **HYPER)
    grads, buf = _tensors(sizes, BF16, cuda_device, 1.0, 8)
    total, coef, lr = (torch.zeros(1, device=cuda_device) for _ in range(3))
    step = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    side = torch.cuda.Stream(device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step.add_(1)
        adamw.grad_norm(grads, total, coef=coef, max_norm=1.0)
        a.step(grads, step=step, lr=lr, coef=coef)
    assert int(step) == 0
    for t in range(1, 6):
        buf.copy_(_tensors(sizes, BF16, cuda_device, float(t), 8 + t)[1])
        lr.fill_(2.0 ** -t)
        graph.replay()
        torch.cuda.synchronize()
        kept = coef.clone()
        adamw.grad_norm(grads, total, coef=coef, max_norm=1.0)
        b.step(grads, step=t, lr=2.0 ** -t, coef=coef)
        torch.cuda.synchronize()
        assert torch.equal(kept, coef) and int(step) == t
        for x, y in zip([*pa, *a.state_dict().values()], [*pb, *b.state_dict().values()]):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.gpu
def test_other_stream(cuda_device):
    params, _ = _tensors([100000], F32, cuda_device, 1.0, 9)
    twin = params[0].clone()
    grads, _ = _tensors([100000], F32, cuda_device, 1.0, 10)
    total, coef = torch.zeros(1, device=cuda_device), torch.zeros(1, device=cuda_device)
    a, b = adamw.AdamW(params, **HYPER), adamw.AdamW([twin], **HYPER)
    side = torch.cuda.Stream(device=cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        adamw.grad_norm(grads, total, coef=coef, max_norm=1.0)
        a.step(grads, step=1, coef=coef)
    side.synchronize()
    adamw.grad_norm(grads, total, coef=coef, max_norm=1.0)
    b.step(grads, step=1, coef=coef)
    assert torch.equal(params[0], twin)


@pytest.mark.gpu
def test_positions_pass_32_bits(cuda_device):
    """One tensor of more than 2^32 elements, 8-bit states: its ends against the definition."""
    n = (1 << 32) + 777
    free, _ = torch.cuda.mem_get_info(cuda_device)
    if free < 60 << 30:
        pytest.skip("needs 60 GiB")
    try:
        p = torch.zeros(n, dtype=BF16, device=cuda_device)
        g = torch.zeros(n, dtype=BF16, device=cuda_device)
        opt = adamw.AdamW([p], state_bits=8, seed=3, **HYPER)
        total, norms = torch.zeros(1, device=cuda_device), torch.zeros(1, device=cuda_device)
        tail = torch.randn(1000).to(BF16)
        g[-1000:] = tail.to(cuda_device)
        adamw.grad_norm([g], total, norms=norms)
        want = tail.double().norm()
        assert abs(float(total) - float(want)) <= 2 * ULP * float(want) and float(norms) == float(total)
        opt.step([g], step=1)
        assert bool((p[:1 << 20] == 0).all()) and bool((p[1 << 31:(1 << 31) + 4096] == 0).all())
        w, m, v, mag, u = _expected(torch.zeros(1000).double(), tail.double(), 0, 0, 1, **HYPER)
        _close(opt.master[n - 1000:n], w, 20 * ULP * u.abs() + 1e-12)
        at = n // 256 * 256  # the last block, 9 elements
        rm, rv = _hash(torch.arange(at, n), 3, 1)
        _check_codes(m[at - n:], mag[at - n:], opt.exp_avg[at:n], opt.exp_avg_scale[-1:], rm, False)
        _check_codes(v.sqrt()[at - n:], v.sqrt()[at - n:], opt.exp_avg_sq[at:n], opt.exp_avg_sq_scale[-1:], rv, True)
    finally:
        p = g = opt = None
        torch.cuda.empty_cache()


# ---- the gradient norm ------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,odd", [([1], False), ([0, 5], False), (SIZES, True), ([3_000_001, 17, 65536], True),
                                       ([(11 * i) % 5000 for i in range(461)], False)])
def test_grad_norm(cuda_device, sizes, odd, dtype):
    grads, _ = _tensors(sizes, dtype, cuda_device, 0.3, len(sizes), odd)
    total, coef, norms = torch.zeros(1, device=cuda_device), torch.zeros(1, device=cuda_device), torch.full((len(sizes),), -1.0, device=cuda_device)
    adamw.grad_norm(grads, total, norms=norms, coef=coef, max_norm=0.7, scale=0.125)
    want = torch.stack([g.double().cpu().square().sum() for g in grads])
    all_of = 0.125 * float(want.sum().sqrt())
    _close(norms, 0.125 * want.sqrt(), 2 * ULP * 0.125 * want.sqrt())
    assert abs(float(total) - all_of) <= 2 * ULP * all_of
    factor = 0.125 * min(1.0, 0.7 / (all_of + 1e-6))
    assert abs(float(coef) - factor) <= 3 * ULP * factor
    again = torch.zeros_like(total)
    adamw.grad_norm(grads, again)
    assert float(again) == pytest.approx(8 * float(total), rel=4 * ULP)


@pytest.mark.gpu
def test_grad_norm_of_extremes(cuda_device):
    """Squares beyond fp32 on either side, missing gradients, zeros, infinities and NaN."""
    total, coef = torch.zeros(1, device=cuda_device), torch.zeros(1, device=cuda_device)

    def of(*grads, **kw):
        adamw.grad_norm(list(grads), total, coef=coef, **kw)
        return float(total), float(coef)

    big = torch.full((1000,), 1e30, device=cuda_device)
    assert of(big, max_norm=1.0)[0] == pytest.approx(1e30 * math.sqrt(1000), rel=1e-6)
    assert of(big * 1e-60, None)[0] == pytest.approx(1e-30 * math.sqrt(1000), rel=1e-6)
    assert of(torch.zeros(9, device=cuda_device), max_norm=1.0) == (0.0, 1.0)
    assert of(None, torch.ones(4, device=cuda_device), scale=0.5) == (1.0, 0.5)
    big[3] = float("inf")
    t, c = of(big, max_norm=1.0)
    assert t == math.inf and math.isnan(c)
    big[4] = float("nan")
    t, c = of(big, max_norm=1.0)
    assert math.isnan(t) and math.isnan(c)


@pytest.mark.gpu
def test_grad_norm_refuses_outputs_that_share_memory(cuda_device):
    b = torch.ones(64, device=cuda_device)
    for total, kw in [(b[:1], dict(coef=b[:1])), (b[3:4], dict(norms=b[2:4])), (b[40:41], {}), (b[:1], dict(norms=b[32:34])),
                      (b[:1], dict(coef=b[63:]))]:
        with pytest.raises(ValueError, match="share memory"):
            adamw.grad_norm([b[40:], b[33:36]], total, **kw)
    adamw.grad_norm([b[40:], b[33:36]], b[:1], norms=b[1:3], coef=b[3:4])
    assert float(b[0]) == pytest.approx(math.sqrt(27), rel=1e-6) and float(b[3]) == 1.0


# ---- together with the norm ---------------------------------------------------------------------
@pytest.mark.gpu
def test_a_training_step_of_all_operators(cuda_device):
    """Partial sums -> residual norm -> loss -> its gradient -> clipped AdamW step on the norm's
    weight, against autograd and the same step in 64 bits."""
    from network_operator_amd.ops import norm

    g = torch.Generator().manual_seed(0)
    xs = [torch.randn(40, 512, generator=g).to(cuda_device) for _ in range(3)]
    res, target = (torch.randn(40, 512, generator=g).to(cuda_device) for _ in range(2))
    w = torch.ones(512, device=cuda_device)
    opt = adamw.AdamW([w], **HYPER)
    out, h, dh = (torch.empty_like(res) for _ in range(3))
    dw = torch.empty_like(w)
    rstd, total, coef = torch.empty(40, device=cuda_device), torch.empty(1, device=cuda_device), torch.empty(1, device=cuda_device)
    norm.add_rms_norm(xs, w, out, residual=res, residual_out=h, rstd=rstd)
    norm.add_rms_norm_backward(out - target, h, w, rstd, dh, dw)
    adamw.grad_norm([dw], total, coef=coef, max_norm=1.0)
    opt.step([dw], step=1, coef=coef)
    w64 = torch.ones(512, dtype=torch.float64, requires_grad=True)
    r64 = res.double().cpu().requires_grad_()
    h64 = sum(x.double().cpu() for x in xs) + r64
    y = h64 * (h64.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w64
    (0.5 * (y - target.double().cpu()).square().sum()).backward()
    assert float((dh.double().cpu() - r64.grad).abs().max()) <= 200 * ULP * float(r64.grad.abs().max() + 4)
    gnorm = float(w64.grad.norm())
    assert abs(float(total) - gnorm) <= 200 * ULP * gnorm
    want = _expected(torch.ones(512).double(), w64.grad * min(1.0, 1.0 / (gnorm + 1e-6)), 0, 0, 1, **HYPER)[0]
    # the first step is lr times the gradient's sign: only where the gradient is no rounding
    clear = w64.grad.abs() > 1e-3
    assert float((w.double().cpu() - want)[clear].abs().max()) <= 1e-6

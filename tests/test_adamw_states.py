"""States, gradients and norms that an optimizer cannot take (ops/adamw.py)."""

import math

import pytest

torch = pytest.importorskip("torch")

from network_operator_amd.ops import adamw  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_states_of_other_sizes_are_refused(cuda_device, bits):
    def opt(*sizes):
        return adamw.AdamW([torch.zeros(n, device=cuda_device) for n in sizes], lr=1e-3, state_bits=bits)

    state = opt(256, 512).state_dict()
    for sizes in [(512, 256), (768,), (250, 512), (256, 511), (256, 256, 256), (256, 0, 512)]:
        with pytest.raises(ValueError, match="sizes"):
            opt(*sizes).load_state_dict(state)
    other = opt(256, 512)
    other.load_state_dict(state)
    other.load_state_dict({k: t for k, t in state.items() if k != "sizes"})  # of a state that was kept without them


def _optimizer(dev, dtype=F32, bits=32):
    buf = torch.zeros(4096, dtype=dtype, device=dev)
    return buf, adamw.AdamW([buf[:600], buf[1000:1300], buf[2000:2005]], lr=1e-2, state_bits=bits)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_in_another_tensors_memory_are_refused(cuda_device, bits):
    buf, opt = _optimizer(cuda_device, BF16, bits)
    g = [torch.ones_like(p) for p in opt.params]
    before = [t.clone() for t in (buf, opt.exp_avg.view(torch.uint8), opt.master)]
    bad = [[opt.params[0], opt.params[0][:300], g[2]], [g[0], buf[900:1200], g[2]], [g[0], buf[1001:1301], g[2]],
           [g[0], g[1], opt.params[1][295:]], [buf[500:1100], g[1], g[2]], [g[0], g[1], buf[2004:2009]], [g[0], None, buf[599:604]]]
    for grads in bad:
        with pytest.raises(ValueError, match="another tensor of this optimizer"):
            opt.step(grads, step=1)
    for t in (opt.master, opt.exp_avg, opt.exp_avg_sq, *(x for x in (opt.exp_avg_scale, opt.exp_avg_sq_scale) if x is not None)):
        with pytest.raises(ValueError, match="another tensor of this optimizer"):  # states, as bf16
            opt.step([g[0], g[1], t.view(torch.uint8)[:10].view(BF16)], step=1)
    with pytest.raises(ValueError, match="another tensor of this optimizer"):
        opt.step(g, step=1, coef=opt.master[:1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (buf, opt.exp_avg.view(torch.uint8), opt.master)))


@pytest.mark.gpu
def test_gradients_in_their_own_parameters_memory(cuda_device):
    for gtype in (BF16, F16):  # two bytes an element as well: read before it is written
        buf, opt = _optimizer(cuda_device, BF16)
        _, ref = _optimizer(cuda_device, BF16)
        for p in opt.params:
            p.fill_(0.5)
        grads = [p.view(gtype) for p in opt.params]
        ref.step([g.clone() for g in grads], step=1)
        opt.step(grads, step=1)
        assert all(torch.equal(p, q) for p, q in zip(opt.params, ref.params))
    _, opt = _optimizer(cuda_device, F32)
    with pytest.raises(ValueError, match="another tensor of this optimizer"):  # half an element: not element on element
        opt.step([p.view(BF16)[:p.numel()] for p in opt.params], step=1)


@pytest.mark.gpu
def test_views_between_the_parameters_are_taken(cuda_device):
    """Gradients right behind and before a parameter, empty ones anywhere, the same one twice."""
    buf = torch.zeros(4096, device=cuda_device)
    opt = adamw.AdamW([buf[0:300], buf[600:900], buf[1000:1000]], lr=1e-2)
    opt.step([buf[300:600], buf[300:600], buf[10:10]], step=1)
    buf[900:1200] = 1
    opt.step([buf[900:1200], buf[900:1200], buf[620:620]], step=2)
    torch.cuda.synchronize()
    assert bool((buf[:300] < 0).all()) and bool((buf[600:900] < 0).all()) and bool((buf[300:600] == 0).all())


@pytest.mark.gpu
def test_a_norm_beyond_fp32_leaves_the_step_out(cuda_device):
    """Finite in 64 bits, infinite as the fp32 total: the factor is NaN, as for any infinite norm."""
    g = torch.full((1000,), 3e38, device=cuda_device)
    total, coef = torch.zeros(1, device=cuda_device), torch.zeros(1, device=cuda_device)
    adamw.grad_norm([g], total, coef=coef, max_norm=1.0)
    assert float(total) == math.inf and math.isnan(float(coef))
    adamw.grad_norm([g], total, coef=coef, max_norm=1.0, scale=2.0 ** -10)
    want = 2.0 ** -10 * float(g[0]) * math.sqrt(1000)
    assert float(total) == pytest.approx(want, rel=2 ** -22) and float(coef) == pytest.approx(2.0 ** -10 / want, rel=1e-6, abs=2e-45)

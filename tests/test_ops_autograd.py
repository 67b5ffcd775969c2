"""The operators and autograd: they write through addresses and are no part of a graph, and say so."""

import pytest

torch = pytest.importorskip("torch")

from network_operator_amd.ops import adamw, norm  # noqa: E402


def _forward(**grad):
    t = {k: torch.zeros(4, 16, requires_grad=grad.get(k, False)) for k in ("x", "residual", "out", "residual_out")}
    w = torch.ones(16, requires_grad=grad.get("weight", False))
    norm.add_rms_norm([t["x"]], w, t["out"], residual=t["residual"], residual_out=t["residual_out"])


@pytest.mark.parametrize("which", ["x", "weight", "residual", "out", "residual_out"])
def test_norm_refuses_what_requires_grad(which):
    with pytest.raises(ValueError, match="automatic differentiation"):
        _forward(**{which: True})
    with torch.no_grad(), pytest.raises(ValueError, match="one CUDA device"):  # the next check
        _forward(**{which: True})


@pytest.mark.parametrize("which", ["dy", "h", "weight", "dresidual", "dh"])
def test_norm_backward_refuses_what_requires_grad(which):
    t = {k: torch.zeros(4, 16, requires_grad=k == which) for k in ("dy", "h", "dh", "dresidual")}
    w = torch.ones(16, requires_grad=which == "weight")

    def call():
        norm.add_rms_norm_backward(t["dy"], t["h"], w, torch.ones(4), t["dh"], torch.zeros(16), dresidual=t["dresidual"])

    with pytest.raises(ValueError, match="automatic differentiation"):
        call()
    with torch.no_grad(), pytest.raises(ValueError, match="one CUDA device"):
        call()


@pytest.mark.gpu
def test_a_graph_that_needs_what_was_overwritten_is_refused(cuda_device):
    """Each output, overwritten after a graph has kept it: its backward pass raises instead of reading the new values."""
    def kept(t):
        return (torch.ones_like(t).requires_grad_() * t).sum()  # the product keeps t

    x, dy = torch.randn(4, 16, device=cuda_device), torch.randn(4, 16, device=cuda_device)
    w, rstd, dw, h, out = (torch.ones(n, device=cuda_device) for n in (16, 4, 16, (4, 16), (4, 16)))
    q, scales = torch.empty(4, 16, dtype=torch.float8_e4m3fn, device=cuda_device), torch.ones(4, device=cuda_device)
    p = [torch.ones(300, device=cuda_device), torch.ones(5, device=cuda_device, dtype=torch.float32)]
    opt = adamw.AdamW(p, lr=0.1)
    total, coef, norms = (torch.ones(n, device=cuda_device) for n in (1, 1, 2))
    g = [torch.ones_like(t) for t in p]
    for written, call in [
        ([out, h, rstd], lambda: norm.add_rms_norm([x], w, out, residual_out=h, rstd=rstd)),
        ([x], lambda: norm.add_rms_norm([x], w, x)),
        ([scales], lambda: norm.add_rms_norm([x], w, q, scales=scales)),
        ([dy, dw], lambda: norm.add_rms_norm_backward(dy, h, w, rstd, dy, dw)),
        ([total, coef, norms], lambda: adamw.grad_norm(g, total, coef=coef, norms=norms)),
        (p + [opt.exp_avg, opt.exp_avg_sq], lambda: opt.step(g, step=1)),
        ([p[1]], lambda: opt.step([None, g[1]], step=2)),
    ]:
        graphs = [kept(t) for t in written]
        call()
        for y in graphs:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    y = kept(p[0])
    opt.step([None, g[1]], step=3)  # left as it was
    y.backward()


@pytest.mark.gpu
def test_tensors_of_inference_mode(cuda_device):
    with torch.inference_mode():
        x, w = torch.randn(4, 16, device=cuda_device), torch.ones(16, device=cuda_device)
        out, p = torch.empty_like(x), torch.ones(16, device=cuda_device)
        norm.add_rms_norm([x], w, out)
        adamw.AdamW([p], lr=0.1).step([w], step=1)
    assert float((out - x * (x.square().mean(1, keepdim=True) + 1e-6).rsqrt()).abs().max()) < 1e-5
    assert abs(float(p[0]) - (1 - 0.1 * 0.01 - 0.1)) < 1e-6

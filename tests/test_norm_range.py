"""The norm's gradient over the whole range of its inputs, against its formula in 64 bits.  Tolerances
are those of tests/test_norm_ops.py: half a step of the output's type, and 80 roundings of the magnitudes
that go into a value."""

import pytest

torch = pytest.importorskip("torch")

from test_norm_ops import BF16, F32, _check_backward  # noqa: E402

from network_operator_amd.ops import norm  # noqa: E402


def _case(shape, dtype, size, dev, seed):
    """h of a root mean square of about ``size``, dy with a part along it, and rstd, as eps = 0 gives it."""
    g = torch.Generator().manual_seed(seed)
    h = (torch.randn(shape, generator=g, dtype=torch.float64) * size).to(dtype).to(dev)
    dy = (torch.randn(shape, generator=g, dtype=torch.float64) * 0.1 + 0.3 * h.cpu().double() / size).to(dtype).to(dev)
    w = (1 + torch.randn(shape[-1], generator=g) * 0.1).to(dtype).to(dev)
    return h, dy, w, h.double().square().mean(-1).rsqrt().float()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-18, 1e-15, 1e-13, 1e14, 1e16, 1e18])
@pytest.mark.parametrize("shape,dtype", [((4, 5), F32), ((5, 40), BF16), ((6, 512), BF16), ((3, 1000), F32), ((3, 4099), BF16),
                                         ((2, 9000), F32), ((2, 20000), BF16), ((2, 32765), F32)])
def test_gradient_of_small_and_large_rows(cuda_device, shape, dtype, size):
    h, dy, w, rstd = _case(shape, dtype, size, cuda_device, shape[1])
    dh, dw = torch.empty_like(h), torch.empty(shape[1], device=cuda_device)
    norm.add_rms_norm_backward(dy, h, w, rstd, dh, dw)
    _check_backward(dy, h, w, rstd, None, dh, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [6, 600, 5003])
def test_gradient_of_a_row_beyond_fp32_is_the_residuals_and_leaves_dweight_alone(cuda_device, cols):
    h, dy, w, _ = _case((5, cols), F32, 1.0, cuda_device, cols)
    h[1] *= 3e37
    dy[1] *= 100
    out, rstd, dres = torch.empty_like(h), torch.empty(5, device=cuda_device), torch.rand_like(h)
    norm.add_rms_norm([h], w, out, rstd=rstd)
    assert float(rstd[1]) == 0 and bool((out[1] == 0).all())
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    norm.add_rms_norm_backward(dy, h, w, rstd, dh, dw, dresidual=dres)
    assert torch.equal(dh[1], dres[1])
    _check_backward(dy, h, w, rstd, dres, dh, dw)

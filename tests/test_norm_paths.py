"""Paths of the norm that depend on size alone: inputs of 64 MiB and more, more rows than one launch
takes, and rows of four vectors a thread over several turns."""

import pytest

torch = pytest.importorskip("torch")

from test_norm_ops import BF16, E4M3, F16, F32, ULP, _check, _check_backward, _close, _empty_like_case, _gradient  # noqa: E402

from network_operator_amd.ops import norm  # noqa: E402


def _randn(shape, dtype, dev, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _forward(xs, w, res, kind):
    out, scales = _empty_like_case(tuple(xs[0].shape), xs[0].dtype, kind, xs[0].device)
    h, rstd = torch.empty(xs[0].shape, dtype=xs[0].dtype, device=xs[0].device), torch.empty(xs[0].shape[0], device=xs[0].device)
    norm.add_rms_norm(xs, w, out, residual=res, residual_out=h, rstd=rstd, scales=scales)
    return [t for t in (out, h, rstd, scales) if t is not None]




def _rows(cols):
    """So many that two inputs of 16 bits are 64 MiB and half of the rows are less, spread over threads alike
    (up to 1024 rows of 8192 are spread wider)."""
    rows = max(-(-(1 << 24) // cols), 2600 if cols == 8192 else 0)
    return rows + rows % 2


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["same", "row", "group"])
@pytest.mark.parametrize("cols", [64, 128, 256, 512, 1024, 4096, 8192, 20000])
def test_forward_of_large_inputs(cuda_device, cols, kind):
    """The same bits as two calls of half the rows (32 MiB), which other tests hold to the definition."""
    rows = _rows(cols)
    dtype = F16 if cols in (128, 4096) else BF16
    x, res = _randn((rows, cols), dtype, cuda_device, cols), _randn((rows, cols), dtype, cuda_device, cols + 1, 2.0)
    w = 1 + _randn(cols, F32, cuda_device, 3, 0.1)
    got = _forward([x], w, res, kind)
    half = rows // 2
    parts = [_forward([x[a:b]], w, res[a:b], kind) for a, b in ((0, half), (half, rows))]
    for t, a, b in zip(got, *parts):
        assert torch.equal(_bits(t), torch.cat([_bits(a), _bits(b)]))
    pick = torch.tensor([0, 1, rows // 2, rows - 1], device=cuda_device)
    out = got[0].view(torch.uint8)[pick].view(E4M3) if kind != "same" else got[0][pick]
    _check([x[pick]], res[pick], w, got[1][pick], got[2][pick], out, got[3][pick] if kind != "same" else None)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 128, 256, 512, 1024, 4096, 8192, 20000])
def test_backward_of_large_inputs(cuda_device, cols):
    rows = _rows(cols)
    dtype = F16 if cols in (128, 4096) else BF16
    dy, h = _randn((rows, cols), dtype, cuda_device, cols, 0.1), _randn((rows, cols), dtype, cuda_device, cols + 1, 2.0)
    w = 1 + _randn(cols, F32, cuda_device, 3, 0.1)
    rstd = h.float().square().mean(1).add(1e-6).rsqrt()
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    norm.add_rms_norm_backward(dy, h, w, rstd, dh, dw)
    half, parts = rows // 2, torch.empty_like(h)
    for a, b in ((0, half), (half, rows)):
        norm.add_rms_norm_backward(dy[a:b], h[a:b], w, rstd[a:b], parts[a:b], torch.empty_like(w))
    assert torch.equal(dh, parts)
    pick = torch.tensor([0, 1, rows // 2, rows - 1], device=cuda_device)
    want, mag, _, _ = _gradient(dy[pick], h[pick], w, rstd[pick], None)
    _close(dh[pick], want, torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + 80 * ULP * mag + torch.finfo(dtype).smallest_normal * 2.0 ** -8)
    terms = dy.double() * h.double() * rstd.double()[:, None]
    # at most a 256th of the rows, then 768 partial rows one after another, three roundings a term
    _close(dw, terms.sum(0).cpu(), (rows / 256 + 768 + 3) * ULP * terms.abs().sum(0).cpu())
    again, dw2 = dy, torch.empty_like(dw)  # in place of dy, the same bits
    norm.add_rms_norm_backward(again, h, w, rstd, again, dw2)
    assert torch.equal(again, dh) and torch.equal(dw2, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("cols,kind", [(5, "same"), (5, "row"), (40, "same"), (40, "row"), (136, "group")])
def test_more_rows_than_a_launch_takes(cuda_device, cols, kind):
    """2^21 rows a launch: the same bits as calls that are cut elsewhere; strided, one row for all among the inputs."""
    rows, cut = (1 << 21) + 5, 1000003
    x = _randn((rows, cols + 3), BF16, cuda_device, 1)[:, 2:2 + cols]
    res = _randn((rows, cols), BF16, cuda_device, 2)
    bias = _randn((1, cols), BF16, cuda_device, 4).expand(rows, cols)
    w = 1 + _randn(cols, F32, cuda_device, 3, 0.1)
    got = _forward([x, bias], w, res, kind)
    parts = [_forward([x[a:b], bias[a:b]], w, res[a:b], kind) for a, b in ((0, cut), (cut, 2 * cut), (2 * cut, rows))]
    for t, *p in zip(got, *parts):
        assert torch.equal(_bits(t), torch.cat([_bits(s) for s in p]))
    pick = torch.tensor([0, (1 << 21) - 1, 1 << 21, rows - 1], device=cuda_device)
    out = got[0].view(torch.uint8)[pick].view(E4M3) if kind != "same" else got[0][pick]
    _check([x[pick], bias[pick]], res[pick], w, got[1][pick], got[2][pick], out, got[3][pick] if kind != "same" else None)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", [(600, 16387, F32), (300, 32765, F32), (300, 32768, F32), (600, 20000, BF16), (270, 16387, F16)])
def test_backward_of_four_vectors_a_thread_over_several_turns(cuda_device, rows, cols, dtype):
    dy, h, dres = (_randn((rows, cols), dtype, cuda_device, k, s) for k, s in ((1, 0.1), (2, 2.0), (3, 0.1)))
    w = (1 + _randn(cols, F32, cuda_device, 4, 0.1)).to(dtype)
    rstd = h.float().square().mean(1).add(1e-6).rsqrt()
    dh, dw = torch.empty_like(h), torch.empty(cols, device=cuda_device)
    norm.add_rms_norm_backward(dy, h, w, rstd, dh, dw, dresidual=dres)
    _check_backward(dy, h, w, rstd, dres, dh, dw)
    for k in range(3):  # in place of dy, h and dresidual: the same bits
        a = [dy.clone(), h.clone(), dres.clone()]
        dw2 = torch.empty_like(dw)
        norm.add_rms_norm_backward(a[0], a[1], w, rstd, a[k], dw2, dresidual=a[2])
        assert torch.equal(a[k], dh) and torch.equal(dw2, dw), k

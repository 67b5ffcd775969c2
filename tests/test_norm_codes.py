"""The norm's e4m3 codes against its own scales, where a value lies at the border of two codes."""

import pytest

torch = pytest.importorskip("torch")

from network_operator_amd.ops import norm  # noqa: E402

F32, E4M3 = torch.float32, torch.float8_e4m3fn
ULP = 2.0 ** -24


def _borders():
    """The values halfway between two codes from 2^-6 up, in 64 bits."""
    codes = torch.arange(8, 127, dtype=torch.uint8).view(E4M3).double()
    return (codes[:-1] + codes[1:]) / 2


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["row", "group"])
@pytest.mark.parametrize("cols", [5, 128, 1000, 8192])
def test_codes_are_nearest_by_the_stored_scale(cuda_device, cols, kind):
    """Rows of ones (rstd = 1), so that the weight is the output: values a few 2^-24 from every border.
    1 / scale and its product with a value are a rounding each: values within 2 * 2^-24 of a border may take
    either code, all others the nearer one; and all are those of value * (1 / scale) in fp32."""
    checked, off = 0, 0
    for seed in range(40):
        g = torch.Generator().manual_seed(seed)
        w = torch.zeros(cols)
        width = cols if kind == "row" else norm.GROUP
        for c in range(0, cols, width):
            n = min(width, cols - c)
            amax = float(torch.rand(1, generator=g) + 1)
            scale = float(torch.tensor(amax) / torch.tensor(448.0))
            b = _borders()[torch.randint(118, (n,), generator=g)]
            off_by = torch.randint(-4, 5, (n,), generator=g).double() * ULP
            w[c:c + n] = (b * scale * (1 + off_by)).float()
            w[c + n - 1] = amax
        w = w.to(cuda_device)
        x = torch.ones(2, cols, device=cuda_device)
        rstd = torch.empty(2, device=cuda_device)
        scales = torch.empty((2,) if kind == "row" else (2, -(-cols // norm.GROUP)), device=cuda_device)
        q = torch.empty(2, cols, dtype=E4M3, device=cuda_device)
        norm.add_rms_norm([x], w, q, scales=scales, rstd=rstd, eps=0.0)
        assert bool((rstd == 1).all())
        per = scales.cpu().double()[1].expand(cols) if kind == "row" else scales.cpu().double()[1].repeat_interleave(norm.GROUP)[:cols]
        u, got = w.cpu().double() / per, q[1].cpu().float().double()
        assert torch.equal(q[1].cpu().view(torch.uint8), (w.cpu() * (1 / per.float())).clamp(max=448).to(E4M3).view(torch.uint8))
        codes = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).double()
        hi = torch.searchsorted(codes, u).clamp(1, 126)
        border = (codes[hi] + codes[hi - 1]) / 2
        sure = (u / border - 1).abs() > 2 * ULP
        want = torch.where(u > border, codes[hi], codes[hi - 1])
        checked += int(sure.sum())
        off += int((got != want)[sure].sum())
        assert bool(((got == codes[hi]) | (got == codes[hi - 1])).all()) and torch.equal(q[0].view(torch.uint8), q[1].view(torch.uint8))
    assert checked > 20 * cols and off == 0

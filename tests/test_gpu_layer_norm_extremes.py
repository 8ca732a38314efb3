"""Layer norm's backward pass at the ends of fp32's range: points of 1e18 and points whose variance is next to nothing."""
import pytest
import torch

from pvn3d_amd.lib import layer_norm as ln

pytestmark = pytest.mark.gpu


def _ref(x, dy, w, mean, rstd):
    """64-bit dx from the statistics that the forward returned (rows)."""
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    u = dy.double() * w.double()
    return rstd.double()[:, None] * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True)), xh, u


@pytest.mark.parametrize("layout", ["rows", "channels"])
@pytest.mark.parametrize("C", [40, 200, 300, 1100, 2100])
@pytest.mark.parametrize("case", ["large", "small"])
def test_gradient_at_the_ends_of_the_range(dev, case, C, layout):
    """C x^2 just within fp32 with small gradients; values of 1e-20 at the smallest variance + eps, with large ones."""
    n = 12
    g = torch.Generator().manual_seed(C)
    x = torch.randn(n, C, generator=g).clamp(-3, 3)
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(dev)
    if case == "large":
        x, eps = x * (8e37 / C) ** 0.5 / 3, 1e-5
        dy = 1e-2 * torch.randn(n, C, generator=g)
    else:
        x, eps = x * 1e-20, 1.5e-38
        dy = 1e4 * (torch.randn(n, C, generator=g) + torch.sign(x))
    x, dy = x.to(dev), dy.to(dev)
    lay = (lambda t: t) if layout == "rows" else (lambda t: t.t().contiguous()[None])
    d = -1 if layout == "rows" else 1
    y, mean, rstd = ln.layer_norm_forward(lay(x), w, None, eps, channel_dim=d)
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(rstd).all()) and float(rstd.min()) > 0
    dx, _, _ = ln.layer_norm_backward(lay(dy), lay(x), w, None, mean, rstd, channel_dim=d)
    got = dx if layout == "rows" else dx[0].t()
    want, xh, u = _ref(x, dy, w, mean, rstd)
    # a mean over C terms is off by 32 roundings of the largest term, xh by four; dx by their sum and its own rounding
    big = rstd.double()[:, None] * u.abs().amax(1, keepdim=True) * (1 + xh.abs().amax(1, keepdim=True) ** 2)
    assert bool(((got.double() - want).abs() <= 32 * 2.0 ** -24 * big).all()), float(((got.double() - want).abs() / big).max())

"""Layer norm (csrc/layer_norm*.hip, lib/layer_norm.py) against its formulas in 64 bits: both layouts, every type, widths
around the kernels' chunk and lane counts, strides, rows with infinities, captured graphs, the 8-bit saved input."""
import pytest
import torch

from pvn3d_amd.lib import act8, layer_norm as ln

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


def _half_step(t):
    return torch.finfo(t).eps / 2


def _ref(x, w, b, relu):
    """64-bit formulas on channels-last data: y, mean, rstd, xh."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPS)
    xh = (x - mean) * rstd
    z = xh * (w.double() if w is not None else 1) + (b.double() if b is not None else 0)
    return (z.clamp_min(0) if relu else z), mean[..., 0], rstd[..., 0], xh


def _ref_grad(dy, xh, rstd, w, on):
    dz = dy.double() * on
    u = dz * (w.double() if w is not None else 1)
    dx = rstd[..., None] * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
    C = xh.size(-1)
    return dx, (dz * xh).reshape(-1, C).sum(0), dz.reshape(-1, C).sum(0)


def _make(shape, C, dt, dev, seed):
    """channels-last x, dy, weight, bias; scale and offset differ by channel."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.linspace(0.3, 2.0, C) + torch.linspace(-1.0, 1.0, C)
    dy = torch.randn(*shape, generator=g)
    w = 1 + 0.3 * torch.randn(C, generator=g)
    b = 0.3 * torch.randn(C, generator=g)
    return x.to(dt).to(dev), dy.to(dt).to(dev), w.to(dev), b.to(dev)


def _amp(x, rstd):
    """How much the rounding of a mean (2^-24 of the point's largest |x|) grows in xh and rstd: 1 + max |x| rstd."""
    return 1 + x.double().abs().amax(-1) * rstd


def _close(got, want, dt, sums=1.0, scale=None):
    """|got - want| <= half a step of the output's type on |want| plus fp32 rounding of the terms: 32 * 2^-24 of `scale`
    (the size of what was added up) times `sums` (the square root of the number of terms beyond the first few)."""
    want = want.double()
    got = got.double()
    scale = scale if scale is not None else want.abs().max().clamp_min(1e-30)
    # fp16: values under 2^-14 are rounded to a multiple of 2^-24
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    bound = _half_step(dt) * want.abs() * (1 + 2.0 ** -10) + 32 * 2.0 ** -24 * sums * scale + tiny
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), "off by %.3g where %.3g is allowed (%d values)" % (
        float(((got - want).abs() - bound).max()), float(bound.min()), int(bad.sum()))


WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 99, 127, 128, 196, 256, 259, 384, 512, 513, 1000, 1024,
          1025, 1536, 2047, 2048, 2049, 4096, 4097, 8192]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_rows_forward_and_backward(dev, C, dt):
    rows = 7 if C > 1024 else 133
    relu = C % 2 == 1
    x, dy, w, b = _make((rows, C), C, dt, dev, C)
    y, mean, rstd = ln.layer_norm_forward(x, w, b, EPS, relu=relu)
    wy, wm, wr, xh = _ref(x, w, b, relu)
    _close(mean, wm, torch.float32, scale=x.double().abs().max())
    # d rstd / rstd = d var / (2 var): relative rounding, and C = 1 has var 0 exactly
    amp = _amp(x, wr)
    assert bool((((rstd.double() - wr) / wr).abs() < 32 * 2.0 ** -24 * amp).all())
    zscale = xh.abs().max() * w.abs().max().double() + b.abs().max().double() + 1e-30
    _close(y, wy, dt, scale=zscale * amp[..., None])
    z = xh * w.double() + b.double()
    on = (z > 0).double() if relu else torch.ones_like(z)
    if relu:        # a value whose sign hangs on rounding gets no gradient
        dy = torch.where(z.abs() < 1e-4 * zscale * amp[..., None], torch.zeros_like(dy), dy)
    dx, dw, db = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu)
    wdx, wdw, wdb = _ref_grad(dy, xh, wr, w, on)
    u = float(dy.abs().max()) * float(w.abs().max())
    _close(dx, wdx, dt, scale=(wr * amp)[..., None] * u * (1 + xh.abs().max() ** 2))
    n = rows ** 0.5
    _close(dw, wdw, torch.float32, n, dy.double().abs().max() * xh.abs().max() * amp.max())
    _close(db, wdb, torch.float32, n, dy.double().abs().max())
    # the same bits again
    again = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu)
    assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), again))
    # one output at a time
    only = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu, need_dparams=False)
    assert only[1] is None and torch.equal(only[0], dx)
    only = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu, need_dx=False)
    assert only[0] is None and torch.equal(only[1], dw) and torch.equal(only[2], db)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,C,M", [(1, 1, 1), (2, 3, 5), (3, 16, 64), (2, 17, 63), (1, 64, 130), (2, 99, 257), (2, 128, 100),
                                   (1, 129, 66), (3, 196, 37), (1, 256, 1), (2, 259, 18), (1, 512, 70), (2, 513, 9),
                                   (1, 1024, 33), (1, 1536, 5), (1, 8192, 3), (5, 8, 1), (0, 8, 4), (2, 8, 0)])
def test_channels_forward_and_backward(dev, B, C, M, dt):
    relu = M % 2 == 1
    x, dy, w, b = _make((B, M, C), C, dt, dev, C + M)
    xc, dyc = x.transpose(1, 2).contiguous(), dy.transpose(1, 2).contiguous()
    y, mean, rstd = ln.layer_norm_forward(xc, w, b, EPS, channel_dim=1, relu=relu)
    assert y.shape == xc.shape and y.is_contiguous() and mean.shape == (B * M,)
    if B * M == 0:
        dx, dw, db = ln.layer_norm_backward(dyc, xc, w, b, mean, rstd, channel_dim=1, relu=relu)
        assert dx.shape == xc.shape and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0
        return
    wy, wm, wr, xh = _ref(x, w, b, relu)
    _close(mean, wm.reshape(-1), torch.float32, scale=x.double().abs().max())
    amp = _amp(x, wr)
    zscale = xh.abs().max() * w.abs().max().double() + b.abs().max().double() + 1e-30
    _close(y.transpose(1, 2), wy, dt, scale=zscale * amp[..., None])
    z = xh * w.double() + b.double()
    on = (z > 0).double() if relu else torch.ones_like(z)
    if relu:
        dyc = torch.where((z.abs() < 1e-4 * zscale * amp[..., None]).transpose(1, 2), torch.zeros_like(dyc), dyc)
    dx, dw, db = ln.layer_norm_backward(dyc, xc, w, b, mean, rstd, channel_dim=1, relu=relu)
    d = dyc.transpose(1, 2)
    wdx, wdw, wdb = _ref_grad(d, xh, wr, w, on)
    u = float(d.abs().max()) * float(w.abs().max())
    _close(dx.transpose(1, 2), wdx, dt, scale=(wr * amp)[..., None] * u * (1 + xh.abs().max() ** 2))
    n = (B * M) ** 0.5
    _close(dw, wdw, torch.float32, n, d.double().abs().max() * xh.abs().max() * amp.max())
    _close(db, wdb, torch.float32, n, d.double().abs().max())
    only = ln.layer_norm_backward(dyc, xc, w, b, mean, rstd, channel_dim=1, relu=relu, need_dx=False)
    assert only[0] is None and torch.equal(only[1], dw) and torch.equal(only[2], db)


@pytest.mark.parametrize("C", [96, 99, 2050])
def test_many_rows_join_their_partial_sums(dev, C):
    """More rows than one pass of the backward grid: several rows per slot, 1024 partial sums."""
    rows = 70001 if C < 1000 else 4099
    x, dy, w, b = _make((rows, C), C, torch.bfloat16, dev, 3)
    y, mean, rstd = ln.layer_norm_forward(x, w, b, EPS)
    dx, dw, db = ln.layer_norm_backward(dy, x, w, b, mean, rstd)
    wy, wm, wr, xh = _ref(x, w, b, False)
    wdx, wdw, wdb = _ref_grad(dy, xh, wr, w, 1.0)
    _close(y, wy, torch.bfloat16)
    _close(dx, wdx, torch.bfloat16, scale=wr.max() * 5 * (1 + xh.abs().max() ** 2))
    _close(dw, wdw, torch.float32, rows ** 0.5, dy.double().abs().max() * xh.abs().max())
    _close(db, wdb, torch.float32, rows ** 0.5, dy.double().abs().max())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,C", [(2048, 1), (2048, 99), (2047, 768), (2049, 1), (2050, 3), (2051, 7), (2060, 8), (2061, 17),
                                    (2061, 33), (4500, 65), (9000, 100), (3001, 259), (2062, 513), (2100, 1000), (2200, 1030),
                                    (1030, 2050), (520, 4100), (300, 8192)])
def test_both_ways_to_the_parameters_gradients(dev, rows, C, dt):
    """Around the border between one launch and partial sums: dx, dweight, dbias from x and from its 8-bit form, in rows of
    a stride of their own."""
    relu = rows % 2 == 1
    x, dy, w, b = _make((rows, C + 3), C + 3, dt, dev, rows + C)
    x, dy, w, b = x[:, :C], dy[:, 2:C + 2], w[:C].contiguous(), b[:C].contiguous()
    wy, wm, wr, xh = _ref(x, w, b, False)
    amp = _amp(x, wr)
    zscale = xh.abs().max() * w.abs().max().double() + b.abs().max().double() + 1e-30
    on = (wy > 0).double() if relu else torch.ones_like(wy)
    if relu:
        dy = torch.where(wy.abs() < 1e-4 * zscale * amp[..., None], torch.zeros_like(dy), dy)
    y, mean, rstd = ln.layer_norm_forward(x, w, b, EPS, relu=relu)
    got = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu)
    u = float(dy.abs().max()) * float(w.abs().max())
    wdx, wdw, wdb = _ref_grad(dy, xh, wr, w, on)
    _close(got[0], wdx, dt, scale=(wr * amp)[..., None] * u * (1 + xh.abs().max() ** 2))
    _close(got[1], wdw, torch.float32, rows ** 0.5, dy.double().abs().max() * xh.abs().max() * amp.max())
    _close(got[2], wdb, torch.float32, rows ** 0.5, dy.double().abs().max())
    again = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu)
    only = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=relu, need_dx=False)
    assert all(torch.equal(p, q) for p, q in zip(got, again)) and torch.equal(only[1], got[1]) and torch.equal(only[2], got[2])
    _, s = ln.layer_norm_forward8(x, w, b, EPS, relu=relu)
    held = act8.act8_unpack(s.act, torch.float32).double()
    xh8 = (held - mean.double()[:, None]) * rstd.double()[:, None]
    got = ln.layer_norm_backward8(dy, s, w)
    if relu:
        on = (((s.mask[:, :, None].int() >> torch.arange(8, device=dev)) & 1).reshape(rows, -1)[:, :C]).double()
    wdx, wdw, wdb = _ref_grad(dy, xh8, rstd.double(), w, on)
    _close(got[0], wdx, dt, scale=rstd.double().max() * u * (1 + xh8.abs().max() ** 2))
    _close(got[1], wdw, torch.float32, rows ** 0.5, dy.double().abs().max() * xh8.abs().max())
    _close(got[2], wdb, torch.float32, rows ** 0.5, dy.double().abs().max())
    only = ln.layer_norm_backward8(dy, s, w, need_dx=False)
    assert torch.equal(only[1], got[1]) and torch.equal(only[2], got[2])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,C,M", [(2, 99, 4095), (1, 3, 8192), (3, 1, 2731), (5, 16, 1700), (1, 40, 8201), (11, 129, 770), (2, 256, 4101),
                                   (2, 300, 4100), (1, 513, 4097), (2, 1024, 1100), (1, 1025, 2100), (3, 2048, 500),
                                   (1, 2049, 1300), (40, 64, 5)])
def test_both_ways_to_the_parameters_gradients_of_channels(dev, B, C, M, dt):
    x, dy, w, b = _make((B, M, C), C, dt, dev, C + M)
    xc, dyc = x.transpose(1, 2).contiguous(), dy.transpose(1, 2).contiguous()
    y, mean, rstd = ln.layer_norm_forward(xc, w, b, EPS, channel_dim=1)
    wy, wm, wr, xh = _ref(x, w, b, False)
    amp = _amp(x, wr)
    zscale = xh.abs().max() * w.abs().max().double() + b.abs().max().double() + 1e-30
    _close(y.transpose(1, 2), wy, dt, scale=zscale * amp[..., None])
    got = ln.layer_norm_backward(dyc, xc, w, b, mean, rstd, channel_dim=1)
    wdx, wdw, wdb = _ref_grad(dy, xh, wr, w, 1.0)
    u = float(dy.abs().max()) * float(w.abs().max())
    _close(got[0].transpose(1, 2), wdx, dt, scale=(wr * amp)[..., None] * u * (1 + xh.abs().max() ** 2))
    n = (B * M) ** 0.5
    _close(got[1], wdw, torch.float32, n, dy.double().abs().max() * xh.abs().max() * amp.max())
    _close(got[2], wdb, torch.float32, n, dy.double().abs().max())
    again = ln.layer_norm_backward(dyc, xc, w, b, mean, rstd, channel_dim=1)
    only = ln.layer_norm_backward(dyc, xc, w, b, mean, rstd, channel_dim=1, need_dx=False)
    assert all(torch.equal(p, q) for p, q in zip(got, again)) and torch.equal(only[1], got[1]) and torch.equal(only[2], got[2])


@pytest.mark.parametrize("dt", TYPES)
def test_strides_and_views(dev, dt):
    g = torch.Generator().manual_seed(1)
    big = torch.randn(40, 3, 70, generator=g).to(dt).to(dev)
    w, b = torch.randn(33, generator=g).to(dev), torch.randn(33, generator=g).to(dev)
    want = ln.layer_norm_forward(big[:, 1, 5:38].contiguous(), w, b)
    got = ln.layer_norm_forward(big[:, 1, 5:38], w, b)                        # strided rows at an odd offset
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and got[0].is_contiguous()
    got = ln.layer_norm_forward(big[:, :, 5:38], w, b)                        # three dimensions, not one row stride apart
    assert torch.equal(got[0][:, 1], want[0]) and got[1].shape == (120,)
    row = big[:1, 0, :33].expand(9, 33)                                       # one row nine times
    y, mean, rstd = ln.layer_norm_forward(row, w, b)
    assert torch.equal(y, y[:1].expand(9, 33)) and torch.equal(y[0], ln.layer_norm_forward(row[0], w, b)[0])
    dy = torch.ones(1, device=dev, dtype=dt).expand(9, 33)                    # gradient of a sum
    d1 = ln.layer_norm_backward(dy, row, w, b, mean, rstd)
    d2 = ln.layer_norm_backward(dy.contiguous(), row.contiguous(), w, b, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(d1, d2))
    # a transposed view of a point-major tensor is read in place and answered in its layout
    pm = torch.randn(2, 50, 33, generator=g).to(dt).to(dev)
    y1, m1, r1 = ln.layer_norm_forward(pm.transpose(1, 2), w, b, channel_dim=1)
    y2, m2, r2 = ln.layer_norm_forward(pm, w, b)
    assert y1.shape == (2, 33, 50) and y1.stride() == pm.transpose(1, 2).stride()
    assert torch.equal(y1.transpose(1, 2), y2) and torch.equal(m1, m2) and torch.equal(r1, r2)
    e = torch.randn(2, 33, 50, generator=g).to(dt).to(dev)
    g1 = ln.layer_norm_backward(e, pm.transpose(1, 2), w, b, m1, r1, channel_dim=1)
    g2 = ln.layer_norm_backward(e.transpose(1, 2).contiguous(), pm, w, b, m1, r1)
    assert torch.equal(g1[0].transpose(1, 2), g2[0]) and torch.equal(g1[1], g2[1]) and torch.equal(g1[2], g2[2])
    # four dimensions, channels second
    x4 = torch.randn(2, 12, 5, 7, generator=g).to(dt).to(dev)
    y4, _, _ = ln.layer_norm_forward(x4, channel_dim=1)
    y3, _, _ = ln.layer_norm_forward(x4.flatten(2), channel_dim=1)
    assert torch.equal(y4.flatten(2), y3)


def test_parameters_may_be_missing(dev):
    x, dy, w, b = _make((65, 40), 40, torch.float32, dev, 9)
    one, zero = torch.ones(40, device=dev), torch.zeros(40, device=dev)
    for ww, bb in ((None, None), (w, None), (None, b)):
        full = (ww if ww is not None else one, bb if bb is not None else zero)
        y, m, r = ln.layer_norm_forward(x, ww, bb, relu=True)
        y2, _, _ = ln.layer_norm_forward(x, *full, relu=True)
        assert torch.equal(y, y2)
        g = ln.layer_norm_backward(dy, x, ww, bb, m, r, relu=True)
        g2 = ln.layer_norm_backward(dy, x, *full, m, r, relu=True)
        assert all(torch.equal(p, q) for p, q in zip(g, g2))
    xc = x.t().contiguous()[None]
    y3, _, _ = ln.layer_norm_forward(xc, None, b, channel_dim=1, relu=True)
    _close(y3[0].t(), _ref(x, None, b, True)[0], torch.float32)


@pytest.mark.parametrize("layout", ["rows", "channels"])
def test_rows_do_not_mix(dev, layout):
    """Infinities and NaN stay in their own point (as torch's formulas have it: the whole point is NaN), the largest finite
    values are normalised, a constant point gives the bias."""
    C, n = 40, 30
    x = torch.randn(n, C, generator=torch.Generator().manual_seed(2))
    x[3, 5], x[7, 0], x[11, 39] = float("inf"), float("-inf"), float("nan")
    x[15] = 2.5
    x[17] *= 1e18
    x = x.to(dev)
    w, b = torch.ones(C, device=dev), torch.full((C,), 0.25, device=dev)
    xin = x if layout == "rows" else x.t().contiguous()[None]
    d = -1 if layout == "rows" else 1
    y, mean, rstd = ln.layer_norm_forward(xin, w, b, channel_dim=d)
    y = y if layout == "rows" else y[0].t()
    bad = [3, 7, 11]
    ok = [i for i in range(n) if i not in bad]
    assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[ok]).all())
    assert torch.equal(y[15], b)
    _close(y[ok], _ref(x[ok], w, b, False)[0], torch.float32)
    dy = torch.ones(n, C, device=dev)
    dyi = dy if layout == "rows" else dy.t().contiguous()[None]
    dx, _, _ = ln.layer_norm_backward(dyi, xin, w, b, mean, rstd, channel_dim=d)
    dx = dx if layout == "rows" else dx[0].t()
    assert bool(torch.isfinite(dx[ok]).all())
    yr, _, _ = ln.layer_norm_forward(xin, w, b, channel_dim=d, relu=True)     # a ReLU passes NaN on
    yr = yr if layout == "rows" else yr[0].t()
    assert bool(torch.isnan(yr[bad]).all())


@pytest.mark.parametrize("channel_dim", [-1, 1])
@pytest.mark.parametrize("relu", [False, True])
def test_gradients_against_differences(dev, channel_dim, relu):
    """Central differences of the call itself in fp32: error h^2 |f'''| / 6 + 2^-24 |f| / h at h = 2^-6."""
    torch.manual_seed(0)
    shape = (3, 5, 9) if channel_dim == 1 else (3, 9, 5)
    m = ln.LayerNorm(5, channel_dim=channel_dim, relu=relu).to(dev)
    with torch.no_grad():
        m.weight.copy_(torch.randn(5))
        m.bias.copy_(torch.randn(5))
    x = (2 * torch.randn(shape)).to(dev).requires_grad_()
    k = torch.randn(shape).to(dev)
    with torch.no_grad():                              # nothing hangs on a value within reach of the ReLU's corner
        z = ln.layer_norm(x, m.weight, m.bias, channel_dim=channel_dim)
        k = torch.where(z.abs() < 0.3, torch.zeros_like(k), k) if relu else k

    def f():
        return (m(x).double() * k).sum()
    f().backward()
    h = 2.0 ** -6
    for p in (x, m.weight, m.bias):
        flat, got = p.data.view(-1), p.grad.reshape(-1)
        for i in range(0, flat.numel(), 7 if p is x else 1):
            v = float(flat[i])
            with torch.no_grad():
                flat[i] = v + h
                up = f()
                flat[i] = v - h
                dn = f()
                flat[i] = v
            want = float(up - dn) / (2 * h)
            assert abs(float(got[i]) - want) < 2e-2 * (1 + abs(want))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", [1, 4, 5, 8, 16, 31, 33, 64, 99, 196, 257, 512, 700, 1025, 2048, 2500, 8192])
def test_saved_in_8_bits(dev, C, dt):
    """forward8's output is forward's; what it keeps is act8_pack(x) and the bits of y > 0; backward8 is the formula with
    the held x."""
    rows = 9 if C > 1024 else 75
    x, dy, w, b = _make((rows, C), C, dt, dev, C + 1)
    for relu in (False, True):
        y, s = ln.layer_norm_forward8(x, w, b, EPS, relu=relu)
        y0, mean, rstd = ln.layer_norm_forward(x, w, b, EPS, relu=relu)
        assert torch.equal(y, y0) and torch.equal(s.mean, mean) and torch.equal(s.rstd, rstd)
        p = act8.act8_pack(x)
        assert torch.equal(s.act.codes, p.codes) and torch.equal(s.act.scales, p.scales)
        held = act8.act8_unpack(p, torch.float32).double()
        xh = (held - mean.double()[:, None]) * rstd.double()[:, None]
        on = torch.ones_like(held)
        if relu:
            bits = (s.mask[:, :, None].int() >> torch.arange(8, device=dev)) & 1
            on = bits.reshape(rows, -1)[:, :C].double()
            z = _ref(x, w, b, False)[0]
            sure = z.abs() > 1e-4 * z.abs().max()
            assert torch.equal(on[sure], (z > 0).double()[sure])
        else:
            assert s.mask is None
        dx, dw, db = ln.layer_norm_backward8(dy, s, w)
        wdx, wdw, wdb = _ref_grad(dy, xh, rstd.double(), w, on)
        u = float(dy.abs().max()) * float(w.abs().max())
        _close(dx, wdx, dt, scale=(rstd.double().max() * u * (1 + xh.abs().max() ** 2)))
        _close(dw, wdw, torch.float32, rows ** 0.5, dy.double().abs().max() * xh.abs().max())
        _close(db, wdb, torch.float32, rows ** 0.5, dy.double().abs().max())
        only = ln.layer_norm_backward8(dy, s, w, need_dx=False)
        assert only[0] is None and torch.equal(only[1], dw)


def test_module_and_autograd(dev):
    """The module's gradients are the functional backward's; ckpt8 holds less memory and works on point-major views; a
    parameter or input without a gradient gets none."""
    x, dy, w, b = _make((4, 300, 64), 64, torch.bfloat16, dev, 5)
    m = ln.LayerNorm(64, relu=True).to(dev)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    xi = x.clone().requires_grad_()
    y = m(xi)
    y.backward(dy)
    y0, mean, rstd = ln.layer_norm_forward(x, w, b, relu=True)
    dx, dw, db = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=True)
    assert torch.equal(y, y0) and torch.equal(xi.grad, dx) and torch.equal(m.weight.grad, dw) and torch.equal(m.bias.grad, db)
    y8, s = ln.layer_norm_forward8(x, w, b, relu=True)
    want = ln.layer_norm_backward8(dy, s, w)
    xi = x.clone().requires_grad_()
    wi, bi = w.clone().requires_grad_(), b.clone().requires_grad_()
    ln.layer_norm(xi, wi, bi, relu=True, ckpt8=True).backward(dy)
    assert all(torch.equal(p, q) for p, q in zip((xi.grad, wi.grad, bi.grad), want))
    xt = x.transpose(1, 2).detach().requires_grad_()
    yt = ln.layer_norm(xt, wi.detach(), bi.detach(), channel_dim=1, relu=True, ckpt8=True)
    yt.backward(dy.transpose(1, 2))
    assert torch.equal(xt.grad.transpose(1, 2), want[0])
    assert s.nbytes < 0.75 * x.numel() * 2
    v = ln.layer_norm(x, wi.detach().requires_grad_(), None)
    v.sum().backward()
    with pytest.raises(RuntimeError):                                          # once only: no second derivative
        xi = x.float().requires_grad_()
        gx, = torch.autograd.grad(ln.layer_norm(xi).sum(), xi, create_graph=True)
        gx.sum().backward()


def test_captured(dev):
    """Forward and backward in one graph, replayed with other inputs and eager work between the replays."""
    C, rows = 99, 513
    x, dy, w, b = _make((rows, C), C, torch.float32, dev, 6)

    def step():
        y, s = ln.layer_norm_forward8(x, w, b, relu=True)
        y2, mean, rstd = ln.layer_norm_forward(x, w, b)
        return (y,) + ln.layer_norm_backward8(dy, s, w) + ln.layer_norm_backward(dy, x, w, b, mean, rstd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(rows, C, generator=torch.Generator().manual_seed(i)))
        dy.copy_(torch.randn(rows, C, generator=torch.Generator().manual_seed(10 + i)))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_more_than_32_bits_of_elements(dev):
    """Row offsets beyond 2^31 elements (a 4.3 GB matrix): first, last and middle rows."""
    rows, C = (1 << 21) + 3, 1032
    x = torch.zeros((rows, C), dtype=torch.bfloat16, device=dev)
    pick = [0, 1, rows // 2, rows - 2, rows - 1]
    g = torch.Generator().manual_seed(4)
    for i in pick:
        x[i] = torch.randn(C, generator=g).to(dev)
    y, mean, rstd = ln.layer_norm_forward(x)
    dx, dw, db = ln.layer_norm_backward(x, x, None, None, mean, rstd)
    s = x[pick]
    ys, ms, rs = ln.layer_norm_forward(s)
    assert torch.equal(y[pick], ys) and torch.equal(mean[pick], ms)
    assert torch.equal(dx[pick], ln.layer_norm_backward(s, s, None, None, ms, rs)[0])


def test_more_than_32_bits_of_channel_rows(dev):
    """(B, C, M) with B C beyond 2^31 (17 GB a tensor): the last clouds as on their own."""
    B, C, M = (1 << 18) + 1, 8192, 4
    x = torch.zeros((B, C, M), dtype=torch.bfloat16, device=dev)
    x[-2:] = torch.randn(2, C, M, generator=torch.Generator().manual_seed(5)).to(dev)
    y, mean, rstd = ln.layer_norm_forward(x, channel_dim=1)
    s = x[-2:].clone()
    ys, ms, rs = ln.layer_norm_forward(s, channel_dim=1)
    assert torch.equal(y[-2:], ys) and torch.equal(mean[-2 * M:], ms) and torch.equal(rstd[-2 * M:], rs)
    del y
    dx = ln.layer_norm_backward(x, x, None, None, mean, rstd, channel_dim=1, need_dparams=False)[0]
    assert torch.equal(dx[-2:], ln.layer_norm_backward(s, s, None, None, ms, rs, channel_dim=1, need_dparams=False)[0])


def test_clouds_of_many_points(dev):
    """More points than the channel-major kernels address: taken as rows."""
    B, C, M = 1, 3, ln.MAX_POINTS + 5
    x = torch.randn(B, C, M, device=dev, generator=torch.Generator("cuda").manual_seed(6))
    w, b = torch.randn(C, device=dev), torch.randn(C, device=dev)
    y, mean, rstd = ln.layer_norm_forward(x, w, b, channel_dim=1)
    yr, mr, rr = ln.layer_norm_forward(x.transpose(1, 2).contiguous(), w, b)
    assert y.is_contiguous() and torch.equal(y, yr.transpose(1, 2)) and torch.equal(mean, mr) and torch.equal(rstd, rr)
    got = ln.layer_norm_backward(x, x, w, b, mean, rstd, channel_dim=1)
    xr = x.transpose(1, 2).contiguous()
    want = ln.layer_norm_backward(xr, xr, w, b, mean, rstd)
    assert torch.equal(got[0], want[0].transpose(1, 2)) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dt,rows,C", [(torch.bfloat16, 690001, 99), (torch.float32, 1050003, 33), (torch.float16, 130007, 601),
                                       (torch.bfloat16, 17000001, 5), (torch.bfloat16, 33001, 2050)])
def test_tensors_larger_than_the_caches(dev, dt, rows, C):
    """Rows of large tensors, which are read and written past the caches, are those of a small one bit for bit."""
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn(rows, C, device=dev, generator=g).to(dt)
    dy = torch.randn(rows, C, device=dev, generator=g).to(dt)
    w, b = torch.randn(C, device=dev, generator=g), torch.randn(C, device=dev, generator=g)
    y, mean, rstd = ln.layer_norm_forward(x, w, b, relu=True)
    dx = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=True, need_dparams=False)[0]
    y8, s = ln.layer_norm_forward8(x, w, b, relu=True)
    dx8 = ln.layer_norm_backward8(dy, s, w, need_dparams=False)[0]
    held = act8.act8_unpack(s.act, dt)
    for i in (0, rows // 2, rows - 1000):
        k = slice(i, i + 1000)
        ys, ms, rs = ln.layer_norm_forward(x[k], w, b, relu=True)
        y8s, ss = ln.layer_norm_forward8(x[k], w, b, relu=True)
        assert torch.equal(y[k], ys) and torch.equal(mean[k], ms) and torch.equal(rstd[k], rs) and torch.equal(y8[k], y8s)
        assert torch.equal(dx[k], ln.layer_norm_backward(dy[k], x[k], w, b, ms, rs, relu=True, need_dparams=False)[0])
        assert torch.equal(dx8[k], ln.layer_norm_backward8(dy[k], ss, w, need_dparams=False)[0])
        assert torch.equal(s.act.codes[k], ss.act.codes) and torch.equal(held[k], act8.act8_unpack(ss.act, dt))


@pytest.mark.parametrize("dt,B,C,M", [(torch.bfloat16, 3, 99, 240001), (torch.float32, 2, 300, 60002), (torch.bfloat16, 2, 1100, 31003),
                                      (torch.float16, 1, 2100, 33001)])
def test_channel_tensors_larger_than_the_caches(dev, dt, B, C, M):
    g = torch.Generator("cuda").manual_seed(M)
    x = torch.randn(B, C, M, device=dev, generator=g).to(dt)
    dy = torch.randn(B, C, M, device=dev, generator=g).to(dt)
    w, b = torch.randn(C, device=dev, generator=g), torch.randn(C, device=dev, generator=g)
    y, mean, rstd = ln.layer_norm_forward(x, w, b, channel_dim=1, relu=True)
    dx = ln.layer_norm_backward(dy, x, w, b, mean, rstd, channel_dim=1, relu=True, need_dparams=False)[0]
    for c, i in ((0, 0), (B - 1, M // 3), (B - 1, M - 1000)):
        k = slice(i, i + 1000)
        xs, ds = x[c:c + 1, :, k].contiguous(), dy[c:c + 1, :, k].contiguous()
        ys, ms, rs = ln.layer_norm_forward(xs, w, b, channel_dim=1, relu=True)
        assert torch.equal(y[c, :, k], ys[0]) and torch.equal(mean.view(B, M)[c, k], ms)
        assert torch.equal(dx[c, :, k], ln.layer_norm_backward(ds, xs, w, b, ms, rs, channel_dim=1, relu=True, need_dparams=False)[0][0])


def test_refusals(dev):
    x = torch.randn(4, 8, device=dev)
    w = torch.ones(8, device=dev)
    m, r = torch.zeros(4, device=dev), torch.ones(4, device=dev)
    bad = [lambda: ln.layer_norm_forward(x.double()), lambda: ln.layer_norm_forward(x, w.half()),
           lambda: ln.layer_norm_forward(x, w[:4]), lambda: ln.layer_norm_forward(x, w.cpu()),
           lambda: ln.layer_norm_forward(x[:, :0]), lambda: ln.layer_norm_forward(torch.randn(2, 8193, device=dev)),
           lambda: ln.layer_norm_forward(torch.randn(2, 3, 4, 5, device=dev), channel_dim=2),
           lambda: ln.layer_norm_backward(x[:2], x, w, w, m, r), lambda: ln.layer_norm_backward(x.half(), x, w, w, m, r),
           lambda: ln.layer_norm_backward(x, x, w, w, m[:2], r), lambda: ln.layer_norm_backward(x, x, w, w, m.double(), r),
           lambda: ln.layer_norm_backward(x, x, w, w, m, r, need_dx=False, need_dparams=False),
           lambda: ln.layer_norm(torch.randn(2, 8, 5, device=dev), channel_dim=1, ckpt8=True),
           lambda: ln.layer_norm_backward8(x, (m, r), w)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("layout", ["rows", "channels"])
def test_on_another_stream(dev, layout):
    x, dy, w, b = _make((2, 700, 128), 128, torch.bfloat16, dev, 8)
    d = -1
    if layout == "channels":
        x, dy, d = x.transpose(1, 2).contiguous(), dy.transpose(1, 2).contiguous(), 1
    y, m, r = ln.layer_norm_forward(x, w, b, channel_dim=d)
    g = ln.layer_norm_backward(dy, x, w, b, m, r, channel_dim=d)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y2, m2, r2 = ln.layer_norm_forward(x, w, b, channel_dim=d)
        g2 = ln.layer_norm_backward(dy, x, w, b, m2, r2, channel_dim=d)
    s.synchronize()
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(g, g2))

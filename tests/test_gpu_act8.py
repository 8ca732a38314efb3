"""The 8-bit form of activations and what is computed from it (csrc/act8.hip, lib/act8.py) against the definition in 64
bits."""
import pytest
import torch

from pvn3d_amd.lib import act8, layer_norm as ln

pytestmark = pytest.mark.gpu


def _held(x):
    """x (rows, C) in the 8-bit form, by the definition: group by group in 64 bits."""
    x = x.double().cpu()
    out = torch.empty_like(x)
    for at in range(0, x.size(1), 32):
        p = x[:, at:at + 32]
        for r in range(p.size(0)):
            big = float(p[r].abs().max())
            if not (big < float("inf")):
                out[r, at:at + 32] = float("nan")
                continue
            e = -126
            while e < 121 and round(big / 2.0 ** e) > 127:
                e += 1
            out[r, at:at + 32] = torch.round(p[r] / 2.0 ** e).clamp(-127, 127) * 2.0 ** e
    return out


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 7), (5, 8), (4, 31), (4, 32), (3, 33), (9, 64), (7, 99), (5, 196), (2, 513),
                                    (3, 1536), (1, 5000)])
def test_held_values_follow_the_definition(dev, rows, C, dt):
    g = torch.Generator().manual_seed(rows * 10000 + C)
    x = torch.randn(rows, C, generator=g) * torch.exp(2 * torch.randn(rows, C, generator=g))
    x[0, 0] = 0.0
    x = x.to(dt)
    act = act8.act8_pack(x.to(dev))
    want = _held(x)
    for out in (torch.float32, torch.bfloat16):
        got = act8.act8_unpack(act, out)
        assert got.dtype == out and got.shape == x.shape and torch.equal(got.double().cpu(), want)   # exact in both
    if dt == torch.float16:
        assert torch.equal(act.unpack(torch.float16).double().cpu(), want)
    groups = [float(x[r, a:a + 32].abs().max()) for r in range(rows) for a in range(0, C, 32)]
    err = [(want[r, a:a + 32] - x[r, a:a + 32].double()).abs().max() for r in range(rows) for a in range(0, C, 32)]
    assert all(float(e) <= m / 127 for e, m in zip(err, groups))              # half a step, a step is at most 2 / 127
    assert act.nbytes == rows * ((C + 15) // 16 * 16 + (C + 31) // 32)


def test_borders(dev):
    """Largest magnitudes next to where the exponent steps, ties, the ends of fp32's range, zeros, non-finite groups."""
    rows = []
    for big in (1.0, 127.0, 127.4999, 127.5, 127.50001, 128.0, 63.75, 63.749996, 2.0 ** -133, 2.0 ** -140, 2.0 ** -149,
                3.4028234e38, 3.3e38, 2.0 ** -126, 2.0 ** -119, 0.0, -0.0):
        r = torch.zeros(32)
        r[0] = big
        r[1:] = torch.linspace(-1, 1, 31) * big
        r[5] = big * 0.5
        rows.append(r)
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.ones(32)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows)
    x = torch.cat([x, torch.ones(x.size(0), 40)], 1)                          # the groups beside a bad one are not touched
    x[-1, 64:] = 3.0
    act = act8.act8_pack(x.to(dev))
    got = act8.act8_unpack(act, torch.float32).double().cpu()
    assert _same(got, _held(x))
    assert bool(torch.isnan(got[-3:, :32]).all()) and bool(torch.isfinite(got[:, 32:]).all())
    assert bool((act.scales[-3:, 0] == 255).all()) and bool((act.codes[-3:, :32] == 0).all())
    assert bool(torch.isnan(act8.act8_unpack(act)[-3:, :32]).all())


def test_strided_input_and_shapes(dev):
    g = torch.Generator().manual_seed(0)
    big = torch.randn(6, 5, 70, generator=g).to(torch.bfloat16).to(dev)
    a = act8.act8_pack(big[:, 2, 3:40])
    b = act8.act8_pack(big[:, 2, 3:40].contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    c = act8.act8_pack(big)
    assert c.shape == big.shape and act8.act8_unpack(c).shape == big.shape and c.codes.shape == (30, 70)
    empty = act8.act8_pack(big[:0])
    assert act8.act8_unpack(empty).shape == (0, 5, 70)
    one = act8.act8_pack(big[0, 0])
    assert act8.act8_unpack(one).shape == (70,)


def _grad_close(dw, dy, held):
    """fp32 sums of exact products: the largest partial sum's rounding, 2^-24 of sum |dy||x| per addition of a chain; the
    chains here are blocked (16 rows a matrix instruction), so 64 roundings of the whole sum's size are far above them."""
    want = dy.double().t() @ held
    size = dy.double().abs().t() @ held.abs()
    assert bool(((dw.double() - want).abs() <= 64 * 2.0 ** -24 * size + 1e-300).all()), \
        float(((dw.double() - want).abs() / size.clamp_min(1e-300)).max())


@pytest.mark.parametrize("rows,M,N", [(1, 1, 1), (31, 8, 8), (32, 32, 32), (33, 33, 33), (100, 64, 32), (127, 32, 64),
                                      (500, 64, 64), (1000, 16, 9), (777, 70, 99), (2049, 128, 128), (300, 129, 257),
                                      (4097, 24, 200), (5000, 200, 24), (64, 512, 1536), (1500, 65, 66), (40, 1, 300),
                                      (40, 300, 1), (65537, 64, 32), (20011, 196, 128), (300, 1000, 40)])
def test_weight_gradient(dev, rows, M, N):
    g = torch.Generator().manual_seed(rows + M + N)
    x = (torch.randn(rows, N, generator=g) * torch.linspace(0.1, 3.0, N)).clamp_min(-0.5).to(torch.bfloat16).to(dev)
    dy = (torch.randn(rows, M, generator=g) * torch.linspace(2.0, 0.5, M)).to(torch.bfloat16).to(dev)
    act = act8.act8_pack(x)
    dw = act8.linear8_weight_grad(dy, act)
    assert dw.shape == (M, N) and dw.dtype == torch.float32
    _grad_close(dw, dy, act8.act8_unpack(act, torch.float32).double())
    assert torch.equal(dw, act8.linear8_weight_grad(dy, act))                 # the same bits
    # strided dy at an odd offset, codes in a wider matrix whose other columns hold anything
    wide = torch.full((rows, M + 13), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 5:5 + M] = dy
    other = torch.randint(-128, 128, (rows, (N + 15) // 16 * 16 + 32), generator=g, dtype=torch.int8).to(dev)
    other[:, :N] = act.codes
    assert torch.equal(dw, act8.linear8_weight_grad(wide[:, 5:5 + M], act8.Act8(other[:, :N], act.scales)))


@pytest.mark.parametrize("rows,M,N", [(100003, 20, 130), (70000, 130, 20), (50001, 200, 300), (33000, 100, 100), (90001, 40, 70),
                                      (1500001, 41, 30), (1400003, 64, 32), (2200000, 20, 50), (2000011, 32, 32)])
def test_weight_gradient_of_many_splits(dev, rows, M, N):
    """Split counts of every tile shape at their largest."""
    test_weight_gradient(dev, rows, M, N)


def test_weight_gradient_of_nothing_and_of_bad_rows(dev):
    dw = act8.linear8_weight_grad(torch.zeros(0, 5, dtype=torch.bfloat16, device=dev),
                                  act8.act8_pack(torch.zeros(0, 7, dtype=torch.bfloat16, device=dev)))
    assert dw.shape == (5, 7) and float(dw.abs().sum()) == 0
    x = torch.ones(50, 70, dtype=torch.bfloat16, device=dev)
    x[3, 40] = float("inf")                                                   # channels 32 .. 63 of one row
    dw = act8.linear8_weight_grad(torch.ones(50, 4, dtype=torch.bfloat16, device=dev), act8.act8_pack(x))
    assert bool(torch.isnan(dw[:, 32:64]).all()) and bool((dw[:, :32] == 50).all()) and bool((dw[:, 64:] == 50).all())


@pytest.mark.parametrize("shape,N", [((100, 64), 32), ((7, 33), 20), ((2, 50, 96), 128), ((4, 5, 9), 16), ((0, 16), 8), ((5,), 3)])
def test_linear8(dev, shape, N):
    """Output and input gradient within a bf16 rounding (and that of the weights) of the fp32 product; the weight's gradient
    is linear8_weight_grad of the kept input; both grads only where wanted."""
    g = torch.Generator().manual_seed(N)
    C = shape[-1]
    x = torch.randn(*shape, generator=g).to(torch.bfloat16).to(dev).requires_grad_()
    w = torch.randn(N, C, generator=g).to(dev).requires_grad_()
    dy = torch.randn(*(shape[:-1] + (N,)), generator=g).to(torch.bfloat16).to(dev)
    y = act8.linear8(x, w)
    assert y.shape == dy.shape and y.dtype == torch.bfloat16
    y.backward(dy)
    wb = w.detach().to(torch.bfloat16).double()
    xd, dd = x.detach().double().reshape(-1, C), dy.double().reshape(-1, N)
    for got, want, size in ((y, xd @ wb.t(), xd.abs() @ wb.abs().t()), (x.grad, dd @ wb, dd.abs() @ wb.abs())):
        got = got.detach().double().reshape(want.shape)
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 64 * 2.0 ** -24 * size).all())
    assert torch.equal(w.grad, act8.linear8_weight_grad(dy, act8.act8_pack(x.detach())))
    if x.numel():
        v = act8.linear8(x.detach(), w)
        v.sum().backward()
        u = act8.linear8(x, w.detach())
        u.sum().backward()


def test_a_layer_and_its_training_pass(dev):
    """convolution -> layer norm -> ReLU -> convolution, everything kept in 8 bits, against the same layers with nothing
    rounded on the way to the backward pass: gradients differ by the 8-bit form alone."""
    g = torch.Generator().manual_seed(11)
    rows, dims = 4000, (64, 96, 32)
    x = torch.randn(rows, dims[0], generator=g).to(torch.bfloat16).to(dev)
    ws = [(torch.randn(b, a, generator=g) / a ** 0.5).to(dev).requires_grad_() for a, b in zip(dims, dims[1:])]
    norm = ln.LayerNorm(dims[1], relu=True, ckpt8=True).to(dev)
    dy = torch.randn(rows, dims[2], generator=g).to(torch.bfloat16).to(dev)
    xi = x.clone().requires_grad_()
    out = act8.linear8(norm(act8.linear8(xi, ws[0])), ws[1])
    out.backward(dy)
    got = [xi.grad, ws[0].grad, ws[1].grad, norm.weight.grad, norm.bias.grad]
    r = [w.detach().to(torch.bfloat16).double().requires_grad_() for w in ws]
    x2 = x.double().requires_grad_()
    nw, nb = norm.weight.detach().double().requires_grad_(), norm.bias.detach().double().requires_grad_()
    h = x2 @ r[0].t()
    h = torch.relu((h - h.mean(1, keepdim=True)) / torch.sqrt(h.var(1, unbiased=False, keepdim=True) + 1e-5) * nw + nb)
    (h @ r[1].t()).backward(dy.double())
    for a, b in zip(got, (x2.grad, r[0].grad, r[1].grad, nw.grad, nb.grad)):
        assert float((a.double() - b).norm() / b.norm()) < 0.03      # bf16 activations (2^-8), steps of 1/64 - 1/128


def test_kept_buffers_are_given_up_behind_the_backward_pass(dev):
    """What a layer keeps goes when its backward pass is done, although the graph's output lives on; a graph that is retained
    can be gone through again; without retaining it a second pass is refused."""
    from pvn3d_amd.lib.layer_norm import layer_norm
    x = torch.randn(4096, 256, device=dev).bfloat16()
    w = torch.randn(256, 256, device=dev, requires_grad=True)
    g = torch.ones(256, device=dev, requires_grad=True)
    b = torch.zeros(256, device=dev, requires_grad=True)
    calls = {"linear8": lambda: act8.linear8(x, w), "layer_norm": lambda: layer_norm(x, g, b, relu=True, ckpt8=True)}
    for name, call in calls.items():
        y = call()
        dy = torch.ones_like(y)
        leaves = [w] if name == "linear8" else [g, b]
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        again = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(first, again)), name
        del first, again
        before = torch.cuda.memory_allocated()
        torch.autograd.grad(y, leaves, dy)
        assert before - torch.cuda.memory_allocated() >= x.numel(), name
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaves, dy)
    # nothing is kept where no gradient is asked for
    before = torch.cuda.memory_allocated()
    y = layer_norm(x, g.detach(), b.detach(), relu=True, ckpt8=True)
    assert torch.cuda.memory_allocated() - before <= 2 * x.numel() and not y.requires_grad


def test_captured(dev):
    g = torch.Generator().manual_seed(12)
    x = torch.randn(700, 99, generator=g).to(torch.bfloat16).to(dev)
    dy = torch.randn(700, 130, generator=g).to(torch.bfloat16).to(dev)

    def step():
        a = act8.act8_pack(x)
        return act8.act8_unpack(a), act8.linear8_weight_grad(dy, a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(700, 99, generator=g))
        dy.copy_(torch.randn(700, 130, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_more_than_32_bits_of_elements(dev):
    """Row offsets beyond 2^31 elements: pack, unpack and the weight gradient of a matrix that is zero but for a few rows."""
    rows, C, M = (1 << 21) + 35, 1032, 24
    x = torch.zeros((rows, C), dtype=torch.bfloat16, device=dev)
    dy = torch.ones((rows, M), dtype=torch.bfloat16, device=dev)
    pick = [0, 1, rows // 2, rows - 33, rows - 2, rows - 1]
    g = torch.Generator().manual_seed(15)
    x[pick] = torch.randn(len(pick), C, generator=g).to(torch.bfloat16).to(dev)
    dy[pick] = torch.randn(len(pick), M, generator=g).to(torch.bfloat16).to(dev)
    act = act8.act8_pack(x)
    held = _held(x[pick])
    out = act8.act8_unpack(act)
    assert torch.equal(out[pick].double().cpu(), held) and int((out != 0).any(1).sum()) == len(pick)
    dw = act8.linear8_weight_grad(dy, act).double().cpu()
    a = dy[pick].double().cpu()
    # six terms and zeros: a rounding of 2^-24 each of the terms' sizes
    assert bool(((dw - a.t() @ held).abs() <= 8 * 2.0 ** -24 * (a.abs().t() @ held.abs())).all())


def test_calls_on_two_streams_at_once(dev):
    """Calls in flight together on two streams share nothing."""
    g = torch.Generator().manual_seed(16)
    sets = []
    for rows, C, M in ((60000, 128, 96), (50001, 99, 70)):
        x = torch.randn(rows, C, generator=g).to(torch.bfloat16).to(dev)
        dy = torch.randn(rows, C, generator=g).to(torch.bfloat16).to(dev)
        d2 = torch.randn(rows, M, generator=g).to(torch.bfloat16).to(dev)
        w, b = torch.rand(C, generator=g).to(dev), torch.rand(C, generator=g).to(dev)
        sets.append((x, dy, d2, w, b))

    def step(x, dy, d2, w, b):
        y, s = ln.layer_norm_forward8(x, w, b, relu=True)
        return (y,) + ln.layer_norm_backward8(dy, s, w) + (act8.linear8_weight_grad(d2, s.act),)
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(r, want[i]))


@pytest.mark.parametrize("dims", [(64, 96, 32), (33, 50, 7)])
def test_a_training_pass_captured(dev, dims):
    """The differentiable calls together, forward and backward in one captured graph, replayed with other inputs."""
    g = torch.Generator().manual_seed(14)
    rows = 1500
    x = torch.zeros(rows, dims[0], dtype=torch.bfloat16, device=dev, requires_grad=True)
    dy = torch.zeros(rows, dims[2], dtype=torch.bfloat16, device=dev)
    ws = [(torch.randn(b, a, generator=g) / a ** 0.5).to(dev).requires_grad_() for a, b in zip(dims, dims[1:])]
    norm = ln.LayerNorm(dims[1], relu=True, ckpt8=True).to(dev)
    leaves = [x] + ws + [norm.weight, norm.bias]

    def step():
        out = act8.linear8(norm(act8.linear8(x, ws[0])), ws[1])
        return (out.detach(),) + torch.autograd.grad(out, leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g))
            dy.copy_(torch.randn(dy.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_refusals(dev):
    x = torch.randn(4, 40, device=dev)
    a = act8.act8_pack(x)
    dy = torch.zeros(4, 8, dtype=torch.bfloat16, device=dev)
    c17 = torch.zeros(4 * 17 + 16, dtype=torch.int8, device=dev)
    bad = [lambda: act8.act8_pack(x.double()), lambda: act8.act8_pack(x[:, :0]), lambda: act8.act8_unpack(x),
           lambda: act8.act8_unpack(a, torch.float64), lambda: act8.linear8_weight_grad(dy.float(), a),
           lambda: act8.linear8_weight_grad(dy[:2], a), lambda: act8.linear8_weight_grad(dy, x),
           lambda: act8.Act8(a.codes, a.scales[:, :1]), lambda: act8.Act8(a.codes.int(), a.scales),
           lambda: act8.Act8(a.codes, a.scales.int()), lambda: act8.Act8(c17[:68].view(4, 17), a.scales[:, :1].contiguous()),
           lambda: act8.Act8(c17[1:65].view(4, 16), a.scales[:, :1].contiguous()),
           lambda: act8.Act8(torch.zeros(4, 40, dtype=torch.int8, device=dev), a.scales),
           lambda: act8.Act8(torch.zeros(17, dtype=torch.int8, device=dev).view(1, 17), a.scales[:1, :1]),
           lambda: act8.Act8(a.codes, a.scales, (2, 2, 39)), lambda: act8.linear8(x, torch.zeros(3, 40, device=dev)),
           lambda: act8.linear8(x.bfloat16(), torch.zeros(3, 39, device=dev)),
           lambda: act8.linear8(x.bfloat16(), torch.zeros(3, 40, device=dev).bfloat16())]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()

"""What ``_train_mlp.ACT_CKPT8`` keeps of the input of a chain: a neighbour's relative coordinates and raw features have a scale
of their own and stay bf16, so their columns of the first weight gradient are those of an unpacked chain."""
import copy

import numpy as np
import pytest
import torch

from pvn3d_amd.lib import act8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,M,K", [(1, 1, 1), (3, 8, 3), (33, 7, 8), (500, 16, 3), (1000, 9, 6), (4099, 64, 3), (70001, 32, 3),
                                      (30000, 128, 6), (100003, 1000, 2), (20011, 196, 8), (1500001, 8, 4), (5000, 260, 5)])
def test_gradient_of_exact_columns(dev, rows, M, K):
    """dy^T x: exact products, fp32 sums in a fixed order.  No chain of additions is longer than 50 rows of a thread, 256
    row slots and 64 partial sums."""
    g = torch.Generator().manual_seed(rows + M + K)
    x = (torch.randn(rows, K, generator=g) * torch.logspace(-2, 2, K)).to(torch.bfloat16).to(dev)
    dy = (torch.randn(rows, M, generator=g) * torch.linspace(2.0, 0.5, M)).to(torch.bfloat16).to(dev)
    dw = act8._columns_weight_grad(dy, x)
    assert dw.shape == (M, K) and dw.dtype == torch.float32
    want, size = dy.double().t() @ x.double(), dy.double().abs().t() @ x.double().abs()
    assert bool(((dw.double() - want).abs() <= 400 * 2.0 ** -24 * size).all())
    assert torch.equal(dw, act8._columns_weight_grad(dy, x))
    wide = torch.full((rows, M + 13), float("nan"), dtype=torch.bfloat16, device=dev)     # rows of a stride, odd offsets
    wide[:, 5:5 + M] = dy
    xw = torch.full((rows, K + 3), float("nan"), dtype=torch.bfloat16, device=dev)
    xw[:, 1:1 + K] = x
    assert torch.equal(dw, act8._columns_weight_grad(wide[:, 5:5 + M], xw[:, 1:1 + K]))


def test_gradient_of_exact_columns_of_nothing_and_refusals(dev):
    z = torch.zeros(0, 5, dtype=torch.bfloat16, device=dev)
    assert float(act8._columns_weight_grad(z, z[:, :3]).abs().sum()) == 0
    dy, x = torch.zeros(4, 5, dtype=torch.bfloat16, device=dev), torch.zeros(4, 9, dtype=torch.bfloat16, device=dev)
    for a, b in ((dy, x), (dy, x[:3, :2]), (dy.float(), x[:, :2]), (dy, x[:, :2].float()), (dy, x[:, :0]), (dy.cpu(), x[:, :2])):
        with pytest.raises(RuntimeError):
            act8._columns_weight_grad(a, b)


def test_gradient_of_exact_columns_beyond_32_bits(dev):
    """Row offsets beyond 2^31 elements: a gradient that is one but for a few rows, columns that are zero but for them."""
    rows, M, K = (1 << 21) + 35, 1032, 3
    dy = torch.ones((rows, M), dtype=torch.bfloat16, device=dev)
    x = torch.zeros((rows, K), dtype=torch.bfloat16, device=dev)
    pick = [0, 1, rows // 2, rows - 33, rows - 2, rows - 1]
    g = torch.Generator().manual_seed(15)
    x[pick] = torch.randn(len(pick), K, generator=g).to(torch.bfloat16).to(dev)
    dy[pick] = torch.randn(len(pick), M, generator=g).to(torch.bfloat16).to(dev)
    dw = act8._columns_weight_grad(dy, x).double()
    a, b = dy[pick].double(), x[pick].double()
    assert bool(((dw - a.t() @ b).abs() <= 8 * 2.0 ** -24 * (a.abs().t() @ b.abs())).all())


def test_gradient_of_exact_columns_captured_and_on_two_streams(dev):
    g = torch.Generator().manual_seed(12)
    sets = [(torch.randn(r, M, generator=g).to(torch.bfloat16).to(dev), torch.randn(r, K, generator=g).to(torch.bfloat16).to(dev))
            for r, M, K in ((60000, 64, 3), (50001, 33, 6))]
    want = [act8._columns_weight_grad(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(act8._columns_weight_grad(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want[i]) for i in range(2) for r in got[i])
    dy, x = sets[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = act8._columns_weight_grad(dy, x)
    for i in range(4):
        dy.copy_(torch.randn(dy.shape, generator=g))
        x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, act8._columns_weight_grad(dy, x))


def _rel(a, b):
    a, b = a.double().flatten(), b.double().flatten()
    return float((a - b).norm() / b.norm())


def _clouds(B, N, dev):
    from pvn3d_amd import synth
    return torch.from_numpy(np.stack([synth.synth_cloud(np.random.default_rng(i), N)[0] for i in range(B)], 0)).to(dev)


def _grads(mod, call, ins, learned, gout, ckpt8):
    """Parameter gradients of a pass through the fused chain; `learned`: which inputs take a gradient."""
    from pvn3d_amd.lib.pointnet2_utils import _train_mlp
    mod = copy.deepcopy(mod)
    ins = [t.clone().detach().requires_grad_(k) for t, k in zip(ins, learned)]
    _train_mlp.TRAIN_FUSED, _train_mlp.ACT_CKPT8 = True, ckpt8
    try:
        out = call(mod, *ins)
        (out.float() * gout).sum().backward()
    finally:
        _train_mlp.TRAIN_FUSED, _train_mlp.ACT_CKPT8 = "auto", False
    return {k: v.grad.detach() for k, v in mod.named_parameters()}


def _cloud_features(B, N, C, dev):
    """(B, C, N): colours 0..255, then unit normals, then more colours."""
    g = torch.Generator().manual_seed(21)
    f = torch.randint(0, 256, (B, C, N), generator=g).float()
    f[:, 3:6] = torch.nn.functional.normalize(torch.randn(B, 3, N, generator=g), dim=1)
    return f.to(dev)


# two fp32 sums of the same exact products in other orders: 400 roundings of 2^-24 of the terms' sizes at most, of which a
# gradient that cancels to 2 % of them leaves 1.2e-3
SAME = 1.2e-3


@pytest.mark.parametrize("norm", ["batch", "layer"])
@pytest.mark.parametrize("learned", [True, False])
def test_coordinates_beside_large_features(dev, norm, learned):
    """A set-abstraction level at the first level's radii with features of 0 .. 255: the coordinates' columns of the first
    layer's weight gradients, and the normals' among raw features."""
    from pvn3d_amd.lib.pointnet2_utils import pointnet2_modules as pm
    torch.manual_seed(3)
    mod = pm.PointnetSAModuleMSG(npoint=256, radii=[0.0175, 0.025], nsamples=[16, 32], mlps=[[6, 16, 32], [6, 32, 64]],
                                 norm=norm).to(dev).train()
    with torch.no_grad():                       # weights of a size that lets every input count
        for name, p in mod.named_parameters():
            if name.endswith("layer0.conv.weight"):
                p[:, :3] *= 5000
                p[:, 6:9] *= 100
    xyz = _clouds(2, 2048, dev)
    f = _cloud_features(2, 2048, 6, dev)
    gout = torch.randn(2, 96, 256, device=dev, generator=torch.Generator("cuda").manual_seed(2))
    call = lambda m, t: m(xyz, t)[1]
    full, kept = (_grads(mod, call, [f], [learned], gout, c) for c in (False, True))
    for k in full:
        if k.endswith("layer0.conv.weight"):
            a, b = kept[k][:, :, 0, 0], full[k][:, :, 0, 0]
            # the layer norm's own input is kept in 8 bits too: its gradient is off by as much as a value of the group
            for cols in (slice(0, 3), slice(3, 6), slice(6, 9)):
                tol = SAME if norm == "batch" else 6.0 / 128
                if learned and cols.start >= 3:
                    # features of a layer: off by 1/128 of the group's largest, 256; colours have an rms of 148, and the
                    # normals share their group, as features of a layer do
                    tol = 6.0 / 128 if cols.start == 3 else None
                if tol is not None:
                    assert _rel(a[:, cols], b[:, cols]) < tol, (k, cols)


@pytest.mark.parametrize("norm", ["batch", "layer"])
def test_raw_features_beside_propagated_ones(dev, norm):
    """A propagation level whose skip features are the cloud's own colours and normals."""
    from pvn3d_amd.lib.pointnet2_utils import pointnet2_modules as pm
    torch.manual_seed(4)
    fp = pm.PointnetFPModule(mlp=[40 + 6, 64, 48], norm=norm).to(dev).train()
    xyz = _clouds(2, 1024, dev)
    known = xyz[:, :256].contiguous()
    g = torch.Generator("cuda").manual_seed(5)
    ins = [_cloud_features(2, 1024, 6, dev), torch.randn(2, 256, 40, device=dev, generator=g).clamp_min(0).transpose(1, 2)]
    gout = torch.randn(2, 48, 1024, device=dev, generator=g)
    call = lambda m, u, k: m(xyz, known, u, k)
    full, kept = (_grads(fp, call, ins, [False, True], gout, c) for c in (False, True))
    for k in full:
        if k.endswith("layer0.conv.weight"):
            a, b = kept[k][:, :, 0, 0], full[k][:, :, 0, 0]
            for cols in (slice(0, 40), slice(40, 43), slice(43, 46)):
                assert _rel(a[:, cols], b[:, cols]) < (SAME if norm == "batch" and cols.start >= 40 else 6.0 / 128), (k, cols)

"""The differentiable layers in front of an operation that changes their output in place (the modules' ReLU does)."""
import pytest
import torch

from pvn3d_amd.lib import act8, layer_norm as ln
from pvn3d_amd.lib.utils import pytorch_utils as pt_utils

pytestmark = pytest.mark.gpu


def _inputs(dev):
    g = torch.Generator().manual_seed(0)
    x4 = torch.randn(2, 12, 5, 7, generator=g).to(dev)
    x3 = torch.randn(3, 50, 12, generator=g).to(dev)
    return {"contiguous": x4, "channels last": x4.to(memory_format=torch.channels_last), "point-major view": x3.transpose(1, 2),
            "one point": x3[:, :1].transpose(1, 2).contiguous(), "three points": x3[:, :3].transpose(1, 2).contiguous()}


@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("kind", ["contiguous", "channels last", "point-major view", "one point", "three points"])
def test_layer_norm(dev, kind, ckpt8):
    x = _inputs(dev)[kind]
    if ckpt8 and kind == "contiguous":
        pytest.skip("channel-major input is refused with ckpt8")
    w, b = torch.rand(12, device=dev), torch.randn(12, device=dev)
    got = []
    for in_place in (False, True):
        p = [t.detach().clone().requires_grad_() for t in (w, b)]
        xi = x.detach().clone().requires_grad_()
        y = ln.layer_norm(xi, *p, channel_dim=1, ckpt8=ckpt8)
        assert y.stride() == ln.layer_norm(xi, *p, channel_dim=1).stride()
        z = torch.relu_(y) if in_place else torch.relu(y)
        (z * torch.linspace(-1, 1, z.numel(), device=dev).view(z.shape)).sum().backward()
        got.append([z.detach(), xi.grad, p[0].grad, p[1].grad])
    assert all(torch.equal(a, c) for a, c in zip(*got))


@pytest.mark.parametrize("shape,N", [((30, 16), 32), ((30, 16), 20), ((2, 15, 33), 7), ((5,), 3)])
def test_linear8(dev, shape, N):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(shape, generator=g).bfloat16().to(dev), torch.randn(N, shape[-1], generator=g).to(dev)
    got = []
    for in_place in (False, True):
        xi, wi = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = act8.linear8(xi, wi)
        z = torch.relu_(y) if in_place else torch.relu(y)
        z.float().sum().backward()
        got.append([z.detach(), xi.grad, wi.grad])
    assert all(torch.equal(a, c) for a, c in zip(*got))


@pytest.mark.parametrize("points", [(1, 1), (1, 2), (4, 8)])
@pytest.mark.parametrize("last", [False, True])
def test_shared_mlp(dev, points, last):
    """SharedMLP(ln=True), whose ReLU works in place, on few points and in the channels-last memory format."""
    torch.manual_seed(0)
    mlp = pt_utils.SharedMLP([6, 8, 5], ln=True).to(dev)
    x = torch.randn(2, 6, *points, device=dev)
    x = x.to(memory_format=torch.channels_last) if last else x
    y = mlp(x.requires_grad_())
    y.sum().backward()
    assert y.shape == (2, 5) + points and all(bool(torch.isfinite(p.grad).all()) for p in mlp.parameters())

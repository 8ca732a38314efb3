"""The ReLU bits that layer_norm_forward8 keeps, byte for byte."""
import pytest
import torch

from pvn3d_amd.lib import layer_norm as ln

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 7, 8, 12, 13, 31, 99, 259, 1030])
@pytest.mark.parametrize("params", [True, False])
def test_bits(dev, dt, C, params):
    """Bit i of byte j is y[8 j + i] > 0, and nothing is set behind the last channel."""
    g = torch.Generator().manual_seed(C)
    x = (torch.randn(40, C, generator=g) - 2).to(dt).to(dev)
    w, b = (torch.randn(C, generator=g).to(dev), torch.randn(C, generator=g).to(dev)) if params else (None, None)
    y, s = ln.layer_norm_forward8(x, w, b, relu=True)
    on = torch.zeros(40, (C + 7) // 8 * 8, dtype=torch.int32, device=dev)
    on[:, :C] = y > 0
    want = (on.view(40, -1, 8) << torch.arange(8, device=dev)).sum(2).to(torch.uint8)
    assert torch.equal(s.mask, want)

"""Points that are not finite through layer norm with its input kept in 8 bits and through the fused training chains: they
reach outputs and gradients as they do op by op."""
import copy

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from pvn3d_amd._lib import check, lib
from pvn3d_amd.lib import layer_norm as ln

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [3, 8, 40, 99, 1030])
def test_a_nan_of_either_sign_passes_the_kept_relu(dev, dt, C):
    """The ReLU's bits of a NaN are on, whatever its sign, so that dx, dweight and dbias have their NaN where the backward
    pass from x has them."""
    g = torch.Generator().manual_seed(C)
    x = torch.randn(12, C, generator=g)
    x[2, C // 2] = float("nan")
    x[5, 0] = torch.tensor([-4194304], dtype=torch.int32).view(torch.float32)[0]           # 0xffc00000
    x[7, C - 1], x[9, 1] = float("inf"), float("-inf")
    x = x.to(dt)
    bits = x.view(torch.int32 if dt == torch.float32 else torch.int16)
    bits[2, C // 2] &= 2 ** 31 - 1 if dt == torch.float32 else 2 ** 15 - 1
    bits[5, 0] |= -2 ** 31 if dt == torch.float32 else -2 ** 15                             # (if a conversion changed it)
    x = x.to(dev)
    dy = torch.randn(12, C, generator=g).to(dt).to(dev)
    dy[5] = float("nan")                                                                   # as an upper layer would hand it on
    w, b = torch.ones(C, device=dev), torch.zeros(C, device=dev)
    y, s = ln.layer_norm_forward8(x, w, b, relu=True)
    on = ((s.mask[:, :, None].int() >> torch.arange(8, device=dev)) & 1).reshape(12, -1)[:, :C].bool()
    assert bool(on[[2, 5, 7, 9]].all()) and torch.equal(on, (y > 0) | torch.isnan(y))
    y0, mean, rstd = ln.layer_norm_forward(x, w, b, relu=True)
    want = ln.layer_norm_backward(dy, x, w, b, mean, rstd, relu=True)
    got = ln.layer_norm_backward8(dy, s, w)
    for p, q in zip(got, want):
        assert torch.equal(torch.isnan(p), torch.isnan(q))

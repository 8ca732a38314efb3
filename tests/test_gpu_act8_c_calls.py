"""The C entry points of the 8-bit form where the Python calls do not go, and which gradients linear8 computes."""
import pytest
import torch

from pvn3d_amd._lib import check, lib
from pvn3d_amd.lib import act8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,t", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)])
@pytest.mark.parametrize("rows,C,ycols,ys", [(1, 1, 16, 16), (5, 3, 4, 7), (40, 33, 48, 64), (77, 64, 64, 64), (300, 99, 112, 113),
                                             (9, 1000, 1008, 1024), (2000, 8, 16, 40)])
def test_unpack_pads_rows(dev, dt, t, rows, C, ycols, ys):
    """Rows of a stride of their own: the held values, zeros in columns C .. y_cols - 1, everything behind them and behind the
    last row as it was."""
    x = torch.randn(rows, C, generator=torch.Generator().manual_seed(C)).to(dt).to(dev)
    act = act8.act8_pack(x)
    out = torch.full((rows * ys + 64,), 7.0, dtype=dt, device=dev)
    codes, scales = act.codes, act.scales
    check(lib.pvn3d_act8_unpack(t, rows, C, codes.data_ptr(), codes.stride(0) if rows > 1 else act.pitch, scales.data_ptr(),
                                out.data_ptr(), ys, ycols, torch.cuda.current_stream().cuda_stream), "act8_unpack")
    m = out[:rows * ys].view(rows, ys)
    assert torch.equal(m[:, :C], act8.act8_unpack(act, dt))
    assert bool((m[:, C:ycols] == 0).all()) and bool((m[:, ycols:] == 7).all()) and bool((out[rows * ys:] == 7).all())


@pytest.mark.parametrize("shape,N", [((100, 64), 32), ((7, 33), 20), ((2, 50, 96), 128), ((5,), 3)])
def test_linear8_only_where_a_gradient_is_asked_for(dev, shape, N):
    g = torch.Generator().manual_seed(N)
    x = torch.randn(*shape, generator=g).to(torch.bfloat16).to(dev)
    w = torch.randn(N, shape[-1], generator=g).to(dev)
    dy = torch.randn(*(shape[:-1] + (N,)), generator=g).to(torch.bfloat16).to(dev)
    xi, wi = x.clone().requires_grad_(), w.clone().requires_grad_()
    act8.linear8(xi, wi).backward(dy)
    x1 = x.clone().requires_grad_()
    act8.linear8(x1, w).backward(dy)
    w1 = w.clone().requires_grad_()
    act8.linear8(x, w1).backward(dy)
    assert torch.equal(x1.grad, xi.grad) and torch.equal(w1.grad, wi.grad)
    assert w.grad is None and x.grad is None
    assert torch.equal(wi.grad, act8.linear8_weight_grad(dy, act8.act8_pack(x)))
    assert not act8.linear8(x, w).requires_grad

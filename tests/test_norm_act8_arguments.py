"""Argument checks that need no GPU, beside those of test_norm_act8_refusals.py."""
import pytest
import torch

from pvn3d_amd._lib import lib
from pvn3d_amd.lib import layer_norm as ln

P = 4096            # a non-null pointer that no refused call may touch


def test_relu_bits_need_a_relu():
    """A mask is the ReLU's: the forward refuses one without it, as the backward does."""
    def call(relu, rows):
        return lib.pvn3d_layer_norm(1, rows, 8, P, 8, None, None, 1e-5, relu, P, 8, 8, P, P, P, 16, P, P, None)
    assert call(0, 4) != 0 and call(0, 0) != 0 and call(1, 0) == 0


def test_exact_columns_refuse():
    ok = dict(rows=4, M=8, K=3, dy=P, dys=8, x=P, xs=3, dw=P, ws=None, wsb=0)

    def call(**kw):
        a = dict(ok, **kw)
        return lib.pvn3d_act8_columns_wgrad(a["rows"], a["M"], a["K"], a["dy"], a["dys"], a["x"], a["xs"], a["dw"], a["ws"],
                                            a["wsb"], None)
    for kw in (dict(K=9), dict(K=-1), dict(M=-1), dict(dys=-1), dict(xs=-1), dict(dys=(1 << 20) + 1), dict(xs=(1 << 20) + 1),
               dict(dy=None), dict(x=None), dict(dw=None), dict(rows=1 << 20), dict(rows=1 << 20, ws=P + 4, wsb=1 << 40),
               dict(rows=1 << 20, ws=P, wsb=64)):
        assert call(**kw) != 0, kw
    assert call(M=0) == 0 and call(K=0) == 0
    assert lib.pvn3d_act8_columns_workspace_bytes(0, 8, 3) == 0 and lib.pvn3d_act8_columns_workspace_bytes(4, 8, 9) == 0
    assert lib.pvn3d_act8_columns_workspace_bytes(1 << 20, 8, 3) % (8 * 3 * 4) == 0


@pytest.mark.parametrize("shape,channel_dim", [((8,), 1), ((8,), 2), ((4, 8), 0), ((4, 8), 3), ((4, 8, 3), -4), ((4, 8, 3, 2), 2),
                                               ((), -1)])
def test_channel_dimensions_that_are_none(shape, channel_dim):
    """A channel_dim that x has not, or that is neither 1 nor the last one, is an error of the call."""
    with pytest.raises(RuntimeError):
        ln._by_rows(torch.zeros(shape), channel_dim)

"""Argument checks of layer norm and the 8-bit activations that need no GPU: the C entry points refuse before they launch,
the Python calls refuse CPU tensors."""
import pytest
import torch

from pvn3d_amd._lib import lib
from pvn3d_amd.lib import act8, layer_norm as ln

P = 4096            # a non-null pointer that no refused call may touch


def test_layer_norm_entry_points_refuse():
    ok = dict(dtype=1, rows=4, C=8, x=P, xs=8, w=None, b=None, eps=1e-5, relu=0, y=P, ys=8, yc=8, mean=P, rstd=P, codes=None,
              pitch=0, scales=None, mask=None)

    def call(**kw):
        a = dict(ok, **kw)
        return lib.pvn3d_layer_norm(a["dtype"], a["rows"], a["C"], a["x"], a["xs"], a["w"], a["b"], a["eps"], a["relu"],
                                    a["y"], a["ys"], a["yc"], a["mean"], a["rstd"], a["codes"], a["pitch"], a["scales"],
                                    a["mask"], None)
    for kw in (dict(dtype=3), dict(dtype=-1), dict(C=0), dict(C=8193), dict(yc=7), dict(yc=24), dict(ys=7), dict(xs=-1),
               dict(x=None), dict(y=None), dict(mean=None), dict(rstd=None), dict(codes=P, pitch=16),
               dict(codes=P, scales=P, pitch=8), dict(codes=P, scales=P, pitch=0), dict(xs=(1 << 20) + 1),
               dict(ys=(1 << 20) + 1)):
        assert call(**kw) != 0, kw
    assert call(rows=0) == 0
    g = dict(dtype=1, rows=100000, C=8, dy=P, dys=8, x=P, xs=8, codes=None, pitch=0, scales=None, mask=None, w=None, b=None, mean=P,
             rstd=P, relu=0, dx=P, dxs=8, dxc=8, dw=P, db=P, ws=P, wsb=1 << 20)

    def grad(**kw):
        a = dict(g, **kw)
        return lib.pvn3d_layer_norm_grad(a["dtype"], a["rows"], a["C"], a["dy"], a["dys"], a["x"], a["xs"], a["codes"],
                                         a["pitch"], a["scales"], a["mask"], a["w"], a["b"], a["mean"], a["rstd"], a["relu"],
                                         a["dx"], a["dxs"], a["dxc"], a["dw"], a["db"], a["ws"], a["wsb"], None)
    for kw in (dict(dtype=4), dict(C=0), dict(C=9000), dict(dys=-1), dict(dxc=7), dict(dxc=24), dict(dxs=4), dict(dw=None),
               dict(db=None), dict(dx=None, dw=None, db=None), dict(x=None), dict(dy=None), dict(mean=None), dict(ws=None),
               dict(wsb=4), dict(codes=P, scales=P, pitch=16, relu=1), dict(codes=P, scales=P, pitch=16, mask=P),
               dict(codes=P, pitch=16), dict(codes=P, scales=P, pitch=4)):
        assert grad(**kw) != 0, kw
    for kw in (dict(dtype=7), dict(B=-1), dict(C=0), dict(M=-1), dict(M=3), dict(M=(1 << 24) + 1), dict(C=8200),
               dict(B=1 << 30, M=1 << 10)):
        a = dict(dict(dtype=0, B=2, C=8, M=4), **kw)
        assert lib.pvn3d_layer_norm_chan(a["dtype"], a["B"], a["C"], a["M"], P, None, None, 1e-5, 0, P, P, P, None) != 0
        assert lib.pvn3d_layer_norm_chan_grad(a["dtype"], a["B"], a["C"], a["M"], P, P, None, None, P, P, 0, P, P, P, P,
                                              1 << 20, None) != 0
    # more points a cloud than the channel slots of them have 32-bit offsets for
    assert lib.pvn3d_layer_norm_chan(0, 1, 2048, (1 << 22) + 1, P, None, None, 1e-5, 0, P, P, P, None) != 0
    assert lib.pvn3d_layer_norm_chan_grad(0, 1, 2048, (1 << 22) + 1, P, P, None, None, P, P, 0, P, P, P, P, 1 << 40, None) != 0
    assert lib.pvn3d_layer_norm_chan_grad(0, 200, 8, 400, P, P, None, None, P, P, 0, P, P, P, None, 0, None) != 0
    assert lib.pvn3d_layer_norm_chan(0, 0, 8, 4, P, None, None, 1e-5, 0, P, P, P, None) == 0
    # the workspace holds a partial dweight and dbias per workgroup
    assert lib.pvn3d_layer_norm_grad_workspace_bytes(1, 10 ** 6, 64) % (2 * 64 * 4) == 0
    assert lib.pvn3d_layer_norm_grad_workspace_bytes(1, 0, 64) == 0
    assert lib.pvn3d_layer_norm_grad_workspace_bytes(1, 100, 64) == 0        # one workgroup: none


def test_act8_entry_points_refuse():
    for a in ((3, 4, 8, P, 8, P, 16, P), (1, 4, 0, P, 8, P, 16, P), (1, 4, 8, P, -1, P, 16, P), (1, 4, 8, P, 8, P, 8, P),
              (1, 4, 17, P, 17, P, 16, P), (1, 4, 8, None, 8, P, 16, P), (1, 4, 8, P, 8, None, 16, P),
              (1, 4, 8, P, 8, P, 16, None)):
        assert lib.pvn3d_act8_pack(*a, None) != 0, a
    for a in ((3, 4, 8, P, 16, P, P, 8, 8), (1, 4, 8, P, 4, P, P, 8, 8), (1, 4, 8, P, 16, P, P, 8, 7),
              (1, 4, 8, P, 16, P, P, 7, 8), (1, 4, 8, P, 16, None, P, 8, 8)):
        assert lib.pvn3d_act8_unpack(*a, None) != 0, a
    for a in ((4, -1, 8, P, 8, P, 16, P, P, None, 0), (4, 8, 8, P, -8, P, 16, P, P, None, 0), (4, 8, 8, P, 8, P, 8, P, P, None, 0),
              (4, 8, 8, None, 8, P, 16, P, P, None, 0), (4, 8, 8, P, 8, P, 16, P, None, None, 0),
              (1 << 20, 8, 8, P, 8, P, 16, P, P, None, 0),                    # row splits without their workspace
              (1 << 20, 8, 8, P, 8, P, 16, P, P, P + 4, 1 << 40)):
        assert lib.pvn3d_act8_wgrad(*a, None) != 0, a
    assert lib.pvn3d_act8_pack(1, 0, 8, None, 8, None, 16, None, None) == 0
    assert lib.pvn3d_act8_wgrad(4, 0, 8, P, 0, P, 16, P, P, None, 0, None) == 0
    assert lib.pvn3d_act8_wgrad_workspace_bytes(0, 8, 8) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for f in (lambda: ln.layer_norm_forward(x), lambda: ln.layer_norm(x), lambda: ln.layer_norm_forward8(x),
              lambda: ln.LayerNorm(8)(x), lambda: ln.layer_norm_backward(x, x, None, None, x[:, 0], x[:, 0]),
              lambda: act8.act8_pack(x), lambda: act8.linear8(x.bfloat16(), torch.zeros(3, 8)),
              lambda: act8.linear8_weight_grad(x.bfloat16(), None),
              lambda: act8.Act8(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8))):
        with pytest.raises(RuntimeError):
            f()

"""Layer norm over the channels of every point, forward and backward (csrc/layer_norm*.hip), beside the BatchNorm that the
SharedMLP layers of the reference use (pvn3d/lib/utils/etw_pytorch_utils/pytorch_utils.py:53-77): the statistics are a
point's own, so a rank that trains on one frame computes what one that trains on 24 does.

    mean = sum_c x / C    var = sum_c (x - mean)^2 / C    rstd = 1 / sqrt(var + eps)    xh = (x - mean) rstd
    y = weight xh + bias, with relu: max(y, 0), NaN where y is

x is float32, bfloat16 or float16; statistics, sums and gradients of the parameters are float32 in a fixed order (the same
bits on every call).  ``channel_dim`` -1: channels last, (..., C), rows of any stride; ``channel_dim`` 1: (B, C, ...), a
contiguous tensor or a transposed view of a point-major one (read in place).  1 <= C <= 8192.  var + eps has to be a normal
fp32 number, 1.2e-38 or more: a point of equal values with eps = 0 is not finite.  A point that holds an infinity or a NaN
is NaN throughout and its statistics are not finite; the other points are not touched by it.

``layer_norm`` is the differentiable call and ``LayerNorm`` the module; ``layer_norm_forward`` / ``layer_norm_backward`` are
the two launches for callers with a backward pass of their own, ``layer_norm_forward8`` / ``layer_norm_backward8`` the same
with the input kept in 8 bits (act8.py) and one bit per value for the ReLU.  Everything runs on the current stream of x's
device and may be captured."""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .._lib import lib, check, on_device
from .act8 import Act8, _dtype, _like, _need, _no_view, _rows, _stream

MAX_CHANNELS = 8192
_CHANNELS = "layer norm takes 1 to %d channels" % MAX_CHANNELS
_F32, _U8 = torch.float32, torch.uint8
MAX_POINTS = 1 << 22         # per cloud, of the channel-major kernels


def _param(p, C, x, name):
    if p is None:
        return None
    if p.dtype is not _F32 or p.dim() != 1 or p.numel() != C:
        raise RuntimeError("%s must be a float32 tensor of the channels' length" % name)
    if p.get_device() != x.get_device():
        raise RuntimeError("%s must be on x's device" % name)
    return p if p.is_contiguous() else p.contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _by_rows(x, channel_dim):
    """-> (True, x with the channels last) or (False, contiguous (B, C, ...)); refuses what is neither."""
    n = x.dim()
    _need(n >= 1, "x must have a channel dimension")
    d = channel_dim + n if channel_dim < 0 else channel_dim
    if d == n - 1:
        rows, C = True, x.size(-1)
    else:
        _need(d == 1 and n > 1, "channel_dim must be 1 or the last dimension")
        C = x.size(1)
        # a point-major view in place; fewer points than a chunk of the channel-major kernel, or more than it addresses:
        # as rows of a copy
        M = x.numel() // max(1, x.size(0) * C)
        rows = not 4 <= M <= MAX_POINTS or (x.movedim(1, -1).is_contiguous() and not x.is_contiguous())
        x = x.movedim(1, -1) if rows else x.contiguous()
    _need(1 <= C <= MAX_CHANNELS, _CHANNELS)
    return rows, x


def _second(y, x):
    """A channels-last result with its channels second, in x's layout: channel-major if x is, else the view it is."""
    y = y.movedim(-1, 1)
    return y.contiguous() if x.is_contiguous() else y


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, channel_dim=-1, relu=False):
    """-> (y like x, mean, rstd): the statistics are float32, one value per point in the points' order."""
    t = _dtype(x, "x")
    rows, v = _by_rows(x, channel_dim)
    C = v.size(-1) if rows else v.size(1)
    w, b = _param(weight, C, x, "weight"), _param(bias, C, x, "bias")
    with on_device(x.device):
        n = v.numel() // C
        y = _like(v)
        mean, rstd = torch.empty(2, n, dtype=_F32, device=x.device).unbind()
        if rows:
            m, xs = _rows(v)
            check(lib.pvn3d_layer_norm(t, n, C, m.data_ptr(), xs, _ptr(w), _ptr(b), eps, 1 if relu else 0, y.data_ptr(), C, C,
                                       mean.data_ptr(), rstd.data_ptr(), None, 0, None, None, _stream(x)), "layer_norm")
            if v is not x:
                y = _second(y, x)
        else:
            check(lib.pvn3d_layer_norm_chan(t, v.size(0), C, n // max(v.size(0), 1), v.data_ptr(), _ptr(w), _ptr(b), eps,
                                            1 if relu else 0, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _stream(x)),
                  "layer_norm_chan")
    return y, mean, rstd


def _grad_buffers(C, wsb, dev):
    """dweight, dbias and the workspace of their partial sums."""
    dw, db = torch.empty(2, C, dtype=_F32, device=dev).unbind()
    ws = torch.empty(wsb, dtype=_U8, device=dev) if wsb else None
    return dw, db, ws, dw.data_ptr(), db.data_ptr(), _ptr(ws)


def _check_stats(mean, rstd, n, x):
    dev = x.get_device()
    for t in (mean, rstd):
        _need(t.dtype is _F32 and t.numel() == n and t.is_contiguous() and t.get_device() == dev,
              "mean and rstd must be contiguous float32 tensors with one value per point")


def layer_norm_backward(dy, x, weight, bias, mean, rstd, channel_dim=-1, relu=False, need_dx=True, need_dparams=True):
    """-> (dx like x or None, dweight (C,), dbias (C,) float32 or None, None).  mean, rstd: the forward's; relu: the
    derivative is 0 where weight xh + bias <= 0 (a NaN passes, as in the forward)."""
    t = _dtype(x, "x")
    _need(dy.shape == x.shape and dy.dtype == x.dtype and dy.get_device() == x.get_device(), "dy must be like x")
    _need(need_dx or need_dparams, "nothing to compute")
    rows, v = _by_rows(x, channel_dim)
    C = v.size(-1) if rows else v.size(1)
    w, b = _param(weight, C, x, "weight"), _param(bias, C, x, "bias")
    n = v.numel() // C
    _check_stats(mean, rstd, n, x)
    dev = x.device
    dx = dw = db = ws = pw = pb = pws = None
    wsb = 0
    with on_device(dev):
        if need_dx:
            dx = _like(v)
        if rows:
            d = dy if v is x else dy.movedim(1, -1)
            (m, xs), (g, gs) = _rows(v), _rows(d)
            if need_dparams:
                wsb = lib.pvn3d_layer_norm_grad_workspace_bytes(t, n, C)
                dw, db, ws, pw, pb, pws = _grad_buffers(C, wsb, dev)
            check(lib.pvn3d_layer_norm_grad(t, n, C, g.data_ptr(), gs, m.data_ptr(), xs, None, 0, None, None, _ptr(w),
                                            _ptr(b), mean.data_ptr(), rstd.data_ptr(), 1 if relu else 0, _ptr(dx), C, C,
                                            pw, pb, pws, wsb, _stream(x)), "layer_norm_grad")
            if need_dx and v is not x:
                dx = _second(dx, x)
        else:
            g = dy.contiguous()
            B = v.size(0)
            M = n // max(B, 1)
            if need_dparams:
                wsb = lib.pvn3d_layer_norm_chan_grad_workspace_bytes(t, B, C, M)
                dw, db, ws, pw, pb, pws = _grad_buffers(C, wsb, dev)
            check(lib.pvn3d_layer_norm_chan_grad(t, B, C, M, g.data_ptr(), v.data_ptr(), _ptr(w), _ptr(b), mean.data_ptr(),
                                                 rstd.data_ptr(), 1 if relu else 0, _ptr(dx), pw, pb, pws, wsb, _stream(x)),
                  "layer_norm_chan_grad")
    return dx, dw, db


class Saved8(object):
    """What layer_norm_forward8 keeps for the backward pass: x in 8 bits (`act`), the statistics `mean` and `rstd`, and with
    a ReLU one bit per value, `mask` (rows, ceil(C / 8)) uint8: bit i of byte j: channel 8 j + i is on (or NaN).  One buffer: codes,
    scales, mask, statistics; views of it are made when they are asked for."""
    __slots__ = ("act", "dtype", "relu", "_buf", "_mask", "_stat")

    def __init__(self, rows, C, shape, dtype, relu, dev, buf=None):
        """buf: an earlier one's buffer."""
        mask = (Act8._bytes(rows, C) + 3) & ~3
        stat = (mask + (rows * ((C + 7) // 8) if relu else 0) + 3) & ~3
        self._buf = torch.empty(stat + 8 * rows, dtype=torch.uint8, device=dev) if buf is None else buf
        self._mask, self._stat, self.dtype, self.relu = mask, stat, dtype, relu
        self.act = Act8._in(self._buf, 0, rows, C, shape)

    def _ptrs(self):
        p = self._buf.data_ptr()
        return p + self._stat, p + self._stat + 4 * self.act.rows, p + self._mask if self.relu else None

    @property
    def mask(self):
        a = self.act
        n = (a.channels + 7) // 8
        return self._buf[self._mask:self._mask + a.rows * n].view(a.rows, n) if self.relu else None

    @property
    def mean(self):
        return self._buf[self._stat:self._stat + 4 * self.act.rows].view(torch.float32)

    @property
    def rstd(self):
        return self._buf[self._stat + 4 * self.act.rows:].view(torch.float32)

    @property
    def nbytes(self):
        return self._buf.numel()


def layer_norm_forward8(x, weight=None, bias=None, eps=1e-5, relu=False):
    """x (..., C) -> (y like x, Saved8).  y is layer_norm_forward's, bit for bit."""
    t = _dtype(x, "x")
    _need(x.dim() >= 1 and 1 <= x.size(-1) <= MAX_CHANNELS, _CHANNELS)
    C = x.size(-1)
    w, b = _param(weight, C, x, "weight"), _param(bias, C, x, "bias")
    dev = x.device
    with on_device(dev):
        m, xs = _rows(x)
        n = x.numel() // C
        y = _like(x)
        saved = Saved8(n, C, x.shape, x.dtype, bool(relu), dev)
        (codes, scales), (mean, rstd, mask) = saved.act._ptrs(), saved._ptrs()
        check(lib.pvn3d_layer_norm(t, n, C, m.data_ptr(), xs, _ptr(w), _ptr(b), eps, 1 if relu else 0, y.data_ptr(), C, C,
                                   mean, rstd, codes, saved.act.pitch, scales, mask, _stream(x)), "layer_norm")
    return y, saved


def layer_norm_backward8(dy, saved, weight=None, need_dx=True, need_dparams=True):
    """layer_norm_backward with xh = (held x - mean) rstd from the 8-bit form and the ReLU from its bits."""
    _need(isinstance(saved, Saved8), "saved must be what layer_norm_forward8 returned")
    t = _dtype(dy, "dy")
    act = saved.act
    _need(dy.shape == act.shape and dy.dtype == saved.dtype and dy.device == act.device, "dy must be like x")
    _need(need_dx or need_dparams, "nothing to compute")
    n, C = act.rows, act.channels
    w = _param(weight, C, dy, "weight")
    dev = dy.device
    dx = dw = db = ws = pw = pb = pws = None
    wsb = 0
    with on_device(dev):
        g, gs = _rows(dy)
        if need_dx:
            dx = _like(dy)
        if need_dparams:
            wsb = lib.pvn3d_layer_norm_grad_workspace_bytes(t, n, C)
            dw, db, ws, pw, pb, pws = _grad_buffers(C, wsb, dev)
        (codes, scales), (mean, rstd, mask) = act._ptrs(), saved._ptrs()
        check(lib.pvn3d_layer_norm_grad(t, n, C, g.data_ptr(), gs, None, 0, codes, act.pitch, scales, mask, _ptr(w), None,
                                        mean, rstd, 1 if saved.relu else 0, _ptr(dx), C, C, pw, pb, pws, wsb, _stream(dy)),
              "layer_norm_grad")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, channel_dim, relu, ckpt8):
        ctx.meta = (channel_dim, relu)
        ctx.kept = None
        if ckpt8:
            rows, v = _by_rows(x, channel_dim)
            _need(rows, "ckpt8 takes channels-last tensors (or a transposed view of one)")
            ctx.moved = v is not x
            if not any(ctx.needs_input_grad):
                y = layer_norm_forward(v, weight, bias, eps, -1, relu)[0]
            else:
                # the buffer as a saved tensor: it is given up behind this layer's backward pass, not with the whole graph
                y, saved = layer_norm_forward8(v, weight, bias, eps, relu)
                ctx.kept = (saved.act.rows, saved.act.channels, saved.act.shape, saved.dtype, saved.relu)
                ctx.save_for_backward(weight, saved._buf)
            return _no_view(_second(y, x) if ctx.moved else y)
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps, channel_dim, relu)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return _no_view(y)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        channel_dim, relu = ctx.meta
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if not (need_x or need_w or need_b):
            return (None,) * 7
        if ctx.kept is not None:
            weight, buf = ctx.saved_tensors
            d = dy.movedim(1, -1) if ctx.moved else dy
            dx, dw, db = layer_norm_backward8(d, Saved8(*ctx.kept, buf.device, buf), weight, need_x, need_w or need_b)
            if ctx.moved and need_x:
                dx = dx.movedim(-1, 1)
        else:
            x, weight, bias, mean, rstd = ctx.saved_tensors
            dx, dw, db = layer_norm_backward(dy, x, weight, bias, mean, rstd, channel_dim, relu, need_x, need_w or need_b)
        return dx, dw if need_w else None, db if need_b else None, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, channel_dim=-1, relu=False, ckpt8=False):
    """Differentiable layer norm (see the top of this file).  ckpt8: keep x for the backward pass in 8 bits instead of
    holding on to it (channels last only); the output is the same, the gradients take xh from the 8-bit form."""
    _dtype(x, "x")
    return _LayerNorm.apply(x, weight, bias, eps, channel_dim, bool(relu), bool(ckpt8) and torch.is_grad_enabled())


class LayerNorm(nn.Module):
    """Layer norm over `channels` channels at `channel_dim` with learned weight (ones) and bias (zeros)."""

    def __init__(self, channels, eps=1e-5, channel_dim=-1, relu=False, ckpt8=False):
        super(LayerNorm, self).__init__()
        self.eps, self.channel_dim, self.relu, self.ckpt8 = eps, channel_dim, relu, ckpt8
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps, self.channel_dim, self.relu, self.ckpt8)

    def extra_repr(self):
        return "%d, eps=%g, channel_dim=%d, relu=%s, ckpt8=%s" % (self.weight.numel(), self.eps, self.channel_dim, self.relu,
                                                                  self.ckpt8)

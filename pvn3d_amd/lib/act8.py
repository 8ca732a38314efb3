"""Activations kept in 8 bits between the forward and the backward pass, and a layer's weight gradient taken from them.

``act8_pack`` / ``act8_unpack``, ``linear8_weight_grad`` and the autograd layer ``linear8`` (the 1x1 convolution of a
SharedMLP layer, ``Conv2d`` of pvn3d/lib/utils/etw_pytorch_utils/pytorch_utils.py:80-134, on point-major rows).  One HIP
launch each, plus one that joins the row splits of a weight gradient (csrc/act8.hip).

The 8-bit form: 32 consecutive channels of a row (the last group of a row may be shorter) share a power of two 2^e and a
value x is held as the int8 code rint(x 2^-e); e >= -126 is the smallest exponent at which the group's largest magnitude
rounds to 127 at most, held as e + 127 in a byte (e <= 121: magnitudes from 127.5 2^121 on are held as 127 2^121).  A value
is off by at most half a step, 1/128 of its group's largest magnitude (half of 2^-126 in a group smaller than that); every
held value is exact in bfloat16.  A group that holds an infinity or a NaN comes back as NaN.
The error is relative to the group: channels much smaller than others of their 32 (coordinates beside features) are held
coarsely or as zeros, and a weight's gradient is lost with its input.  Such columns do not belong in this form.

Everything runs on the current stream of the tensors' device and reads only its arguments; calls may be captured."""
import torch
from torch.autograd.function import once_differentiable

from .._lib import lib, check, on_device

GROUP = 32
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# torch.cuda.current_stream() builds a Stream object: 1.9 us a call more than torch's own short cut, where there is one
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _stream(t):
    return _raw_stream(t.get_device())


def _need(ok, what):
    if not ok:
        raise RuntimeError(what)


def _dtype(t, name):
    """The kernels' number of t's type; refuses CPU tensors and other types."""
    _need(t.is_cuda, "CPU not supported")
    d = DTYPES.get(t.dtype)
    if d is None:
        raise RuntimeError("%s must be a float32, bfloat16 or float16 tensor" % name)
    return d


MAX_STRIDE = 1 << 20        # row strides (in elements) that the kernels take; wider ones are copied


def _rows(t):
    """(..., C) -> (a tensor that starts with its rows -- t itself, a 2-D view or a copy, channels contiguous --, the rows'
    stride)."""
    C = t.size(-1)
    if t.is_contiguous():
        return t, C
    m = t if t.dim() == 2 else t.reshape(-1, C)
    if (m.stride(1) != 1 and C > 1) or m.stride(0) > MAX_STRIDE:
        m = m.contiguous()
    return m, (m.stride(0) if m.size(0) > 1 else C)


def _like(m):
    """An uninitialised contiguous tensor of m's type and shape."""
    return torch.empty_like(m) if m.is_contiguous() else m.new_empty(m.shape)


def _no_view(t):
    """t's memory as a tensor that is no view: an output of an autograd function that is one cannot be changed in place, as a
    ReLU(inplace=True) behind the layer does."""
    if not t._is_view():
        return t
    return torch.empty(0, dtype=t.dtype, device=t.device).set_(t.untyped_storage(), t.storage_offset(), t.size(), t.stride())


def _align16(n):
    return (n + 15) & ~15


class Act8(object):
    """A tensor (..., C) in the 8-bit form: `codes` int8 (rows, C), rows 16-byte aligned (pitch a multiple of 16, whole
    16-byte chunks in its storage), `scales` uint8 (rows, ceil(C / 32)) contiguous, `shape` of the tensor."""
    __slots__ = ("_codes", "_scales", "_buf", "_at", "rows", "channels", "pitch", "shape", "device")

    def __init__(self, codes, scales, shape=None):
        _need(codes.dtype is torch.int8 and codes.dim() == 2, "codes must be an int8 matrix")
        rows, C = size = codes.shape
        _need(C > 0, "codes must have at least one channel")
        _need(scales.dtype is torch.uint8 and scales.shape == (rows, (C + GROUP - 1) // GROUP)
              and scales.is_contiguous(), "scales must be a contiguous uint8 (rows, ceil(channels / 32)) matrix")
        _need(codes.is_cuda and scales.is_cuda, "CPU not supported")
        _need(scales.get_device() == codes.get_device(), "scales must be on the codes' device")
        pitch = _align16(C)
        if rows > 0:
            step, inner = codes.stride()
            _need((inner == 1 or C == 1) and codes.data_ptr() % 16 == 0
                  and (rows == 1 or (step % 16 == 0 and C <= step <= MAX_STRIDE)), "codes must have 16-byte aligned rows")
            last = codes.storage_offset() + (rows - 1) * step + pitch
            _need(codes.untyped_storage().nbytes() >= last, "codes must end with a whole 16-byte chunk")
            if rows > 1:
                pitch = step
        if shape is not None:
            n = 1
            for v in shape[:-1]:
                n *= v
            _need(len(shape) > 0 and shape[-1] == C and n == rows, "shape does not fit the codes")
            size = torch.Size(shape)
        self._codes, self._scales, self._buf, self._at = codes, scales, None, 0
        self.rows, self.channels, self.pitch, self.shape, self.device = rows, C, pitch, size, codes.device

    @staticmethod
    def _in(buf, at, rows, C, shape):
        """The codes from byte `at` (a multiple of 16) of a uint8 buffer on, the scales behind them; views of it are made
        when they are asked for."""
        act = object.__new__(Act8)
        act._codes = act._scales = None
        act._buf, act._at, act.rows, act.channels, act.pitch, act.shape = buf, at, rows, C, _align16(C), shape
        act.device = buf.device
        return act

    @staticmethod
    def _bytes(rows, C):
        return rows * (_align16(C) + (C + GROUP - 1) // GROUP)

    @property
    def codes(self):
        if self._codes is None:
            n = self.rows * self.pitch
            self._codes = self._buf[self._at:self._at + n].view(torch.int8).view(self.rows, self.pitch)[:, :self.channels]
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            at, G = self._at + self.rows * self.pitch, (self.channels + GROUP - 1) // GROUP
            self._scales = self._buf[at:at + self.rows * G].view(self.rows, G)
        return self._scales

    def _ptrs(self):
        if self._buf is not None:
            p = self._buf.data_ptr() + self._at
            return p, p + self.rows * self.pitch
        return self._codes.data_ptr(), self._scales.data_ptr()

    @property
    def nbytes(self):
        return self.rows * (self.pitch + (self.channels + GROUP - 1) // GROUP)

    def unpack(self, dtype=torch.bfloat16):
        return act8_unpack(self, dtype)


def act8_pack(x):
    """x (..., C) float32 / bfloat16 / float16 -> Act8."""
    t = _dtype(x, "x")
    C = x.size(-1) if x.dim() else 0
    _need(C > 0, "x must have at least one channel")
    dev = x.device
    with on_device(dev):
        m, xs = _rows(x)
        rows = x.numel() // C
        act = Act8._in(torch.empty(Act8._bytes(rows, C), dtype=torch.uint8, device=dev), 0, rows, C, x.shape)
        codes, scales = act._ptrs()
        check(lib.pvn3d_act8_pack(t, rows, C, m.data_ptr(), xs, codes, act.pitch, scales, _stream(x)), "act8_pack")
    return act


def act8_unpack(act, dtype=torch.bfloat16):
    """Act8 -> the held values, a contiguous tensor of its shape.  bfloat16 and float32 hold every value exactly; float16
    does if the tensor was a float16 one (otherwise values are rounded, and overflow to infinity)."""
    _need(isinstance(act, Act8), "act must be an Act8")
    t = DTYPES.get(dtype)
    _need(t is not None, "dtype must be float32, bfloat16 or float16")
    dev = act.device
    with on_device(dev):
        out = torch.empty(*act.shape, dtype=dtype, device=dev)
        codes, scales = act._ptrs()
        check(lib.pvn3d_act8_unpack(t, act.rows, act.channels, codes, act.pitch, scales, out.data_ptr(), act.channels,
                                    act.channels, _stream(out)), "act8_unpack")
    return out


def linear8_weight_grad(dy, act):
    """dW (M, N) float32 = dy^T X: dy (..., M) bfloat16, X the rows of `act` (..., N).  Exact operands, fp32 sums in a fixed
    order (the same bits on every call); no rows: zeros."""
    _need(dy.is_cuda, "CPU not supported")
    _need(dy.dtype is torch.bfloat16, "dy must be a bfloat16 tensor")
    _need(isinstance(act, Act8), "act must be an Act8")
    dev = dy.device
    _need(act.device == dev, "act must be on dy's device")
    rows, N, M = act.rows, act.channels, dy.size(-1) if dy.dim() else 0
    _need(M > 0, "dy must have at least one channel")
    _need(dy.numel() == rows * M, "dy and act must have the same number of rows")
    with on_device(dev):
        m, ds = _rows(dy)
        dw = torch.empty(M, N, dtype=torch.float32, device=dev)
        wsb = lib.pvn3d_act8_wgrad_workspace_bytes(rows, M, N)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        codes, scales = act._ptrs()
        check(lib.pvn3d_act8_wgrad(rows, M, N, m.data_ptr(), ds, codes, act.pitch, scales, dw.data_ptr(),
                                   ws.data_ptr() if wsb else None, wsb, _stream(dy)), "act8_wgrad")
    return dw


MAX_COLUMNS = 8             # of _columns_weight_grad


def _columns_weight_grad(dy, x):
    """dW (M, K) float32 = dy^T x for a few columns that are kept in bfloat16 beside the codes: dy (rows, M), x (rows, K),
    K <= 8, both bfloat16.  fp32 sums in a fixed order, like linear8_weight_grad."""
    _need(dy.is_cuda and x.device == dy.device, "x must be on dy's device")
    _need(dy.dtype is torch.bfloat16 and x.dtype is torch.bfloat16, "dy and x must be bfloat16 tensors")
    _need(dy.dim() == 2 and x.dim() == 2 and dy.size(0) == x.size(0), "dy and x must have the same number of rows")
    rows, M, K, dev = dy.size(0), dy.size(1), x.size(1), dy.device
    _need(M > 0 and 0 < K <= MAX_COLUMNS, "dy must have at least one channel, x 1 to %d" % MAX_COLUMNS)
    with on_device(dev):
        (m, ds), (v, xs) = _rows(dy), _rows(x)
        dw = torch.empty(M, K, dtype=torch.float32, device=dev)
        wsb = lib.pvn3d_act8_columns_workspace_bytes(rows, M, K)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        check(lib.pvn3d_act8_columns_wgrad(rows, M, K, m.data_ptr(), ds, v.data_ptr(), xs, dw.data_ptr(),
                                           ws.data_ptr() if wsb else None, wsb, _stream(dy)), "act8_columns_wgrad")
    return dw


def _ld(c):
    return (int(c) + 15) // 16 * 16


def _padded(m, C):
    """(rows, C) bfloat16 -> (matrix whose rows hold a multiple of 16 channels, zeros behind C, 16-byte aligned; its row
    stride): what the matrix kernel reads."""
    if (C % 16 == 0 and m.stride(1) == 1 and m.data_ptr() % 16 == 0
            and (m.size(0) <= 1 or (m.stride(0) % 8 == 0 and C <= m.stride(0) < 2 ** 31))):
        return m, (m.stride(0) if m.size(0) > 1 else C)
    out = torch.zeros((m.size(0), _ld(C)), dtype=torch.bfloat16, device=m.device)
    out[:, :C] = m
    return out, _ld(C)


def _product(m, C, weight, transpose):
    """rows x weight^T (transpose = False: weight (N, C)) or rows x weight (weight (C, N)), bfloat16 (rows, N), the rows
    padded to a multiple of 16 channels in memory."""
    N = weight.size(1) if transpose else weight.size(0)
    dev, st = m.device, _stream(m)
    out = torch.empty((m.size(0), _ld(N)), dtype=torch.bfloat16, device=dev)
    if m.size(0):
        a, lda = _padded(m, C)
        ldw = _ld(C)
        wb = torch.empty((N, ldw), dtype=torch.bfloat16, device=dev)
        check(lib.pvn3d_mt_pack_weight(weight.size(0), weight.size(1), weight.data_ptr(), weight.size(1),
                                       1 if transpose else 0, wb.data_ptr(), N, ldw, st), "mt_pack_weight")
        check(lib.pvn3d_mt_gemm_nt(m.size(0), N, ldw, a.data_ptr(), lda, wb.data_ptr(), ldw, out.data_ptr(), _ld(N),
                                   None, None, 0, st), "mt_gemm_nt")
    return out if out.size(1) == N else out[:, :N]


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, keep):
        N, C = weight.shape
        with on_device(x.device):
            w = weight.detach().contiguous()
            y = _product(x.reshape(-1, C), C, w, False)
            buf = ctx.kept = None
            if keep and ctx.needs_input_grad[1]:
                act = act8_pack(x.detach())
                ctx.kept, buf = (act.rows, C, act.shape), act._buf
        ctx.save_for_backward(weight, buf)        # (the buffer is given up behind this layer's backward pass)
        ctx.lead = x.shape[:-1]
        return _no_view(y.view(x.shape[:-1] + (N,)) if x.dim() != 2 else y)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, buf = ctx.saved_tensors
        N, C = weight.shape
        dx = dw = None
        dy = dy.to(torch.bfloat16)
        with on_device(dy.device):
            m = dy.reshape(-1, N)
            if ctx.needs_input_grad[0]:
                dx = _product(m, N, weight.detach().contiguous(), True).reshape(ctx.lead + (C,))
            if ctx.needs_input_grad[1]:
                dw = linear8_weight_grad(m, Act8._in(buf, 0, *ctx.kept))
        return dx, dw, None


def linear8(x, weight):
    """y (..., N) = x (..., C) weight^T on the bfloat16 matrix kernels, x bfloat16, weight (N, C) float32 (rounded to
    bfloat16 for the product, like the fused training chain does).  x is kept for the backward pass in 8 bits; the
    input's gradient does not depend on it, the weight's is taken from it.  y's rows may be padded in memory (N not a
    multiple of 16)."""
    _need(x.is_cuda, "CPU not supported")
    _need(x.dtype == torch.bfloat16, "x must be a bfloat16 tensor")
    _need(weight.device == x.device, "weight must be on x's device")
    _need(weight.dim() == 2 and weight.dtype == torch.float32, "weight must be a float32 matrix")
    _need(x.dim() >= 1 and x.size(-1) == weight.size(1) and weight.numel() > 0, "x and weight must have the same channels")
    _need(x.numel() // x.size(-1) < 2 ** 31, "too many rows")
    return _Linear8.apply(x, weight, torch.is_grad_enabled())

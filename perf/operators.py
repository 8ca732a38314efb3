"""Layer norm, 8-bit activation checkpoints and the weight gradient taken from them: the calls that are timed, their plain
forms in elementary torch operations, and their values in 64 bits.

A training step of the voting branch runs [1x1 convolution -> norm -> ReLU] on point-major matrices, one row per (cloud,
centre, neighbour); the sizes below are those of its levels at 24 frames of 12288 points, and of single frames.
"""
import math

import torch

own = False

EPS = 1e-5
GROUP = 32                      # channels of a row that share one scale of the 8-bit form
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the deepest level of one frame: a call whose cost is its launch
        dict(name="ln_fwd_one_frame", op="ln_fwd", layout="rows", rows=128, c=512, dtype="bf16", relu=True),
        # features as the modules hand them over, channel-major, 24 whole clouds
        dict(name="ln_fwd_clouds_fp32", op="ln_fwd", layout="channels", rows=24 * 12288, b=24, c=128, dtype="fp32", relu=False),
        # first set-abstraction level, wide scale: 24 clouds x 2048 centres x 32 neighbours
        dict(name="ln_fwd_level0_bf16", op="ln_fwd", layout="rows", rows=24 * 2048 * 32, c=64, dtype="bf16", relu=True),
        # relative coordinates ++ 96 features: an odd width, full precision
        dict(name="ln_bwd_odd_fp32", op="ln_bwd", layout="rows", rows=10007, c=99, dtype="fp32", relu=False),
        # grouped tensors (B, C, npoint, nsample) of the op-by-op composition
        dict(name="ln_bwd_grouped_bf16", op="ln_bwd", layout="channels", rows=8 * 512 * 32, b=8, c=196, dtype="bf16", relu=True),
        # second level, 128 wide
        dict(name="ln_bwd_level1_bf16", op="ln_bwd", layout="rows", rows=24 * 1024 * 32, c=128, dtype="bf16", relu=True),
        # a whole pass over a layer that keeps its input in 8 bits: third level, ragged last group of channels
        dict(name="ln_train8_level2_bf16", op="ln_train8", layout="rows", rows=24 * 512 * 32, c=196, dtype="bf16", relu=True),
        # the same for one frame of a propagation level
        dict(name="ln_train8_one_frame_fp16", op="ln_train8", layout="rows", rows=512, c=512, dtype="fp16", relu=True),
        # a chain's input put away for the backward pass and fetched again
        dict(name="act8_level1_bf16", op="act8", layout="rows", rows=24 * 1024 * 32, c=96, dtype="bf16", relu=False),
        # coordinates ++ 256 features, full precision
        dict(name="act8_odd_fp32", op="act8", layout="rows", rows=6007, c=259, dtype="fp32", relu=False),
        # weight gradient of a narrow layer over many rows
        dict(name="wgrad8_level0", op="wgrad8", layout="rows", rows=24 * 2048 * 32, c=32, m=64, dtype="bf16", relu=True),
        # weight gradient of the widest layer
        dict(name="wgrad8_widest", op="wgrad8", layout="rows", rows=24 * 512, c=1536, m=512, dtype="bf16", relu=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "ln_train8", "act8", "wgrad8"])
    if op == "wgrad8":
        m, c = _log(rng, 8, 512), _log(rng, 8, 1536)
        most = min(24 * 2048 * 32, 9.0e9 / (m * c), 1.0e8 / (m + c))
        return dict(op=op, layout="rows", rows=_log(rng, 64, most), c=c, m=m, dtype="bf16", relu=True)
    c = _log(rng, 8, 1536)
    rows = _log(rng, 64, min(24 * 2048 * 32, 3.5e7 / c))
    case = dict(op=op, layout="rows", rows=rows, c=c, dtype=rng.choice(["fp32", "bf16", "fp16"]), relu=rng.random() < 0.5)
    if op in ("ln_fwd", "ln_bwd") and rng.random() < 0.4:
        b = rng.randint(1, 24)
        case.update(layout="channels", b=b, rows=max(1, rows // b) * b)
    if op == "act8":
        case["relu"] = False
    return case


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, c, t = case["rows"], case["c"], TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("wgrad8", "act8"):
        # activations: channels of different scale; behind a ReLU about half of them are zero
        x = _randn(g, rows, c) * (0.25 + 2.0 * torch.rand(c, generator=g, device="cuda")) + 0.2 * _randn(g, c)
        x = (x.clamp_min(0) if case["relu"] else x).to(t)
        if case["op"] == "act8":
            s["x"] = x
            return s
        codes, scales = _codes(x)
        pitch = (c + 15) // 16 * 16
        s["codes"] = torch.zeros(rows, pitch, dtype=torch.int8, device="cuda")[:, :c]
        s["codes"].copy_(codes)
        s["scales"] = scales
        s["dy"] = (_randn(g, rows, case["m"]) * 1e-2).to(t)
        return s
    shape = (rows, c) if case["layout"] == "rows" else (case["b"], c, rows // case["b"])
    per = (c,) if case["layout"] == "rows" else (1, c, 1)
    # outputs of a convolution: channels of different scale and offset
    x = _randn(g, *shape) * (0.3 + torch.rand(*per, generator=g, device="cuda")) + 0.3 * _randn(g, *per)
    s["x"] = x.to(t)
    s["weight"] = 1.0 + 0.2 * _randn(g, c)
    s["bias"] = 0.2 * _randn(g, c)
    if case["op"] == "ln_fwd":
        return s
    dy = _randn(g, *shape) * 1e-2
    y, mean, rstd = _ln_fwd(s["x"].float(), s["weight"], s["bias"], per, _dim(case))
    if case["relu"]:
        # a value whose sign hangs on its last bits gets no gradient: either side of the ReLU is right for it
        dy = torch.where(y.abs() < 1e-4, torch.zeros_like(dy), dy)
    s["dy"] = dy.to(t)
    if case["op"] == "ln_bwd":
        s["mean"], s["rstd"] = mean.reshape(-1), rstd.reshape(-1)
    return s


def _dim(case):
    return 1


def _per(case):
    return (case["c"],) if case["layout"] == "rows" else (1, case["c"], 1)


def _ln_fwd(x, weight, bias, per, dim):
    mean = x.mean(dim, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(dim, keepdim=True) + EPS)
    return d * rstd * weight.view(per) + bias.view(per), mean, rstd


def _ln_bwd(dz, xh, rstd, weight, per, dim):
    u = dz * weight.view(per)
    dx = rstd * (u - u.mean(dim, keepdim=True) - xh * (u * xh).mean(dim, keepdim=True))
    over = [d for d in range(dz.dim()) if d != dim]
    return dx, (dz * xh).sum(over), dz.sum(over)


def _in_groups(x):
    rows, c = x.shape
    n = (c + GROUP - 1) // GROUP
    if n * GROUP == c:
        return x.reshape(rows, n, GROUP)
    full = torch.zeros(rows, n * GROUP, dtype=x.dtype, device=x.device)
    full[:, :c] = x
    return full.view(rows, n, GROUP)


def _codes(x):
    """x (rows, c) -> int8 codes (rows, c) and the biased exponents (rows, ceil(c / 32)) of their groups' powers of two:
    the smallest exponent, -126 at least, at which the group's largest magnitude rounds to 127 at most."""
    g = _in_groups(x.float())
    big = g.abs().amax(2, keepdim=True)
    fine = torch.isfinite(big)
    frac, e = torch.frexp(torch.where(fine, big, torch.zeros_like(big)))
    e = torch.clamp(e - 7 + (torch.round(frac * 128) > 127).int(), min=-126)
    q = torch.round(torch.ldexp(g, -e))
    q = torch.where(fine, q, torch.zeros_like(q)).to(torch.int8)
    scales = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return q.reshape(x.size(0), -1)[:, :x.size(1)], scales[:, :, 0]


def _values(codes, scales):
    two = torch.where(scales == 255, torch.full_like(scales, float("nan"), dtype=torch.float32),
                      torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127))
    return (_in_groups(codes.float()) * two[:, :, None]).reshape(codes.size(0), -1)[:, :codes.size(1)]


def run(s):
    case = s["case"]
    op, relu = case["op"], case["relu"]
    if own:
        from pvn3d_amd.lib import act8, layer_norm
        d = -1 if case["layout"] == "rows" else 1
        if op == "ln_fwd":
            return layer_norm.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS, channel_dim=d, relu=relu)
        if op == "ln_bwd":
            return layer_norm.layer_norm_backward(s["dy"], s["x"], s["weight"], s["bias"], s["mean"], s["rstd"],
                                                  channel_dim=d, relu=relu)
        if op == "ln_train8":
            y, saved = layer_norm.layer_norm_forward8(s["x"], s["weight"], s["bias"], EPS, relu=relu)
            return (y,) + tuple(layer_norm.layer_norm_backward8(s["dy"], saved, s["weight"]))
        if op == "act8":
            return act8.act8_unpack(act8.act8_pack(s["x"]))
        return act8.linear8_weight_grad(s["dy"], act8.Act8(s["codes"], s["scales"]))

    if op == "act8":
        return _values(*_codes(s["x"])).to(torch.bfloat16)
    if op == "wgrad8":
        return s["dy"].float().t() @ _values(s["codes"], s["scales"])
    per, dim, t = _per(case), _dim(case), s["x"].dtype
    x = s["x"].float()
    if op == "ln_bwd":
        stat = (x.size(0), 1) if case["layout"] == "rows" else (x.size(0), 1, x.size(2))
        mean, rstd = s["mean"].view(stat), s["rstd"].view(stat)
        xh = (x - mean) * rstd
        dz = s["dy"].float()
        if relu:
            dz = dz * (xh * s["weight"].view(per) + s["bias"].view(per) > 0)
        dx, dw, db = _ln_bwd(dz, xh, rstd, s["weight"], per, dim)
        return dx.to(t), dw, db
    z, mean, rstd = _ln_fwd(x, s["weight"], s["bias"], per, dim)
    y = (z.clamp_min(0) if relu else z).to(t)
    if op == "ln_fwd":
        return y, mean.reshape(-1), rstd.reshape(-1)
    dz = s["dy"].float()
    if relu:
        dz = dz * (z > 0)
    dx, dw, db = _ln_bwd(dz, (_values(*_codes(s["x"])) - mean) * rstd, rstd, s["weight"], per, dim)
    return y, dx.to(t), dw, db


def work(case):
    rows, c, op = case["rows"], case["c"], case["op"]
    e, n = TYPES[case["dtype"]].itemsize, case["rows"] * case["c"]
    groups = rows * ((c + GROUP - 1) // GROUP)
    if op == "ln_fwd":
        return {"bytes": 2 * n * e + 8 * rows + 8 * c, "flops": 8 * n}
    if op == "ln_bwd":
        return {"bytes": 3 * n * e + 8 * rows + 16 * c, "flops": 14 * n}
    if op == "ln_train8":       # x, y, dy and dx; the 8-bit copy and the mask are written and read again
        return {"bytes": 4 * n * e + 2 * (n + groups) + (n // 4 if case["relu"] else 0) + 24 * c, "flops": 26 * n}
    if op == "act8":
        return {"bytes": n * e + 2 * (n + groups) + 2 * n, "flops": 5 * n}
    return {"bytes": 2 * rows * case["m"] + n + groups + 4 * case["m"] * c, "flops": 2 * n * case["m"]}


def exact(case, seed):
    s = prepare(case, seed)
    op, relu = case["op"], case["relu"]

    def eighth(x):
        """Every value of x (rows, c) to the nearest multiple of its group's step (ties to the even multiple), in 64 bits."""
        out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        for at in range(0, x.size(1), GROUP):
            part = x[:, at:at + GROUP].double()
            big = part.abs().max(1, keepdim=True).values
            step = torch.exp2(torch.floor(torch.log2(big.clamp_min(2.0 ** -120))) - 6)
            step = torch.where(torch.round(big / step) > 127, 2 * step, step).clamp_min(2.0 ** -126)
            out[:, at:at + GROUP] = torch.round(part / step) * step
        return out

    if op == "act8":
        return eighth(s["x"])
    if op == "wgrad8":
        step = torch.exp2(s["scales"].double() - 127.0).repeat_interleave(GROUP, 1)[:, :case["c"]]
        x, dy = s["codes"].double() * step, s["dy"].double()
        total = torch.zeros(case["m"], case["c"], dtype=torch.float64, device=x.device)
        for at in range(0, case["rows"], 1 << 17):
            total += torch.matmul(dy[at:at + (1 << 17)].t(), x[at:at + (1 << 17)])
        return total

    # rows first: (b, c, n) -> (b n, c), and back for what is laid out like x
    flat = (lambda v: v) if case["layout"] == "rows" else (lambda v: v.transpose(1, 2).reshape(-1, case["c"]))
    back = (lambda v: v) if case["layout"] == "rows" else \
        (lambda v: v.view(case["b"], -1, case["c"]).transpose(1, 2).contiguous())
    x, w, b = flat(s["x"].double()), s["weight"].double(), s["bias"].double()
    if op == "ln_bwd":
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
    else:
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = torch.rsqrt(var + EPS)
    z = torch.addcmul(b, (x - mean) * rstd, w)
    y = torch.relu(z) if relu else z
    if op == "ln_fwd":
        return back(y), mean[:, 0], rstd[:, 0]
    dz = flat(s["dy"].double())
    if relu:
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    xh = ((eighth(s["x"]) if op == "ln_train8" else x) - mean) * rstd
    u = dz * w
    n = float(case["c"])
    dx = rstd * (u - u.sum(1, keepdim=True) / n - xh * ((u * xh).sum(1, keepdim=True) / n))
    grads = (back(dx), torch.einsum("rc,rc->c", dz, xh), dz.sum(0))
    return ((back(y),) + grads) if op == "ln_train8" else grads

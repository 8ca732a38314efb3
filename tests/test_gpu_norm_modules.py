"""Layer norm and 8-bit kept activations where the framework's modules use them: SharedMLP in SA / FP modules with
norm="layer" (op by op and the fused bf16 chain), and ``_train_mlp.ACT_CKPT8`` with either norm."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rel(a, b):
    a, b = a.double().flatten(), b.double().flatten()
    return float((a - b).norm() / max(float(b.norm()), 1e-12))


def _clouds(B, N, dev):
    from pvn3d_amd import synth
    return torch.from_numpy(np.stack([synth.synth_cloud(np.random.default_rng(i), N)[0] for i in range(B)], 0)).to(dev)


def _sa(dev, norm):
    from pvn3d_amd.lib.pointnet2_utils import pointnet2_modules as pm
    torch.manual_seed(3)
    mod = pm.PointnetSAModuleMSG(npoint=128, radii=[0.05, 0.1], nsamples=[16, 32],
                                 mlps=[[10, 16, 32], [10, 32, 24, 64]], norm=norm).to(dev).train()
    for p in mod.parameters():
        if p.dim() == 1:
            p.data.uniform_(0.5, 1.5)
    return mod


def _run(mod, call, inputs, gout, fused, ckpt8=False, autocast=False):
    from pvn3d_amd.lib.pointnet2_utils import _train_mlp
    mod = copy.deepcopy(mod)
    ins = [t.clone().detach().requires_grad_(True) for t in inputs]
    _train_mlp.TRAIN_FUSED, _train_mlp.ACT_CKPT8 = fused, ckpt8
    try:
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autocast(device_type="cuda", dtype=torch.bfloat16, enabled=autocast):
            out = call(mod, *ins)
        held = torch.cuda.memory_allocated() - before
        (out.float() * gout).sum().backward()
    finally:
        _train_mlp.TRAIN_FUSED, _train_mlp.ACT_CKPT8 = "auto", False
    return dict(out=out.detach().float(), ins=[t.grad.detach() for t in ins], held=held,
                params={k: v.grad.detach() for k, v in mod.named_parameters()})


def _cases(dev, norm):
    """(module, call, inputs, gradient of the output) of an SA level and of an FP module."""
    from pvn3d_amd.lib.pointnet2_utils import pointnet2_modules as pm
    xyz = _clouds(2, 1024, dev)
    feats = torch.randn(2, 1024, 10, device=dev, generator=torch.Generator("cuda").manual_seed(1)).transpose(1, 2)
    yield (_sa(dev, norm), lambda m, f: m(xyz, f)[1], [feats],
           torch.randn(2, 96, 128, device=dev, generator=torch.Generator("cuda").manual_seed(2)))
    torch.manual_seed(4)
    fp = pm.PointnetFPModule(mlp=[40 + 7, 64, 48], norm=norm).to(dev).train()
    for p in fp.parameters():
        if p.dim() == 1:
            p.data.uniform_(0.5, 1.5)
    known = xyz[:, :256].contiguous()
    g = torch.Generator("cuda").manual_seed(5)
    yield (fp, lambda m, u, k: m(xyz, known, u, k),
           [torch.randn(2, 7, 1024, device=dev, generator=g), torch.randn(2, 256, 40, device=dev, generator=g).transpose(1, 2)],
           torch.randn(2, 48, 1024, device=dev, generator=g))


@pytest.mark.parametrize("which", [0, 1])
def test_layer_norm_modules_op_by_op(dev, which):
    """fp32, no autocast: the composition with the layer-norm kernel in it against the same weights through torch's own
    operations in fp64."""
    mod, call, ins, gout = list(_cases(dev, "layer"))[which]
    got = _run(mod, call, ins, gout, fused=False)

    class TorchNorm(torch.nn.Module):
        def __init__(self, ln):
            super().__init__()
            self.weight, self.bias, self.eps = ln.weight, ln.bias, ln.eps

        def forward(self, x):
            x64 = x.double()
            mean = x64.mean(1, keepdim=True)
            y = (x64 - mean) / torch.sqrt(((x64 - mean) ** 2).mean(1, keepdim=True) + self.eps)
            shape = (1, -1) + (1,) * (x.dim() - 2)
            return (y * self.weight.double().view(shape) + self.bias.double().view(shape)).float()
    ref = copy.deepcopy(mod)
    for m in list(ref.modules()):
        if hasattr(m, "ln"):
            m.ln = TorchNorm(m.ln)
    want = _run(ref, call, ins, gout, fused=False)
    # forward: fp32 convolutions on both sides.  Gradients: a ReLU or a maximum that hangs on the last bits goes another way
    # for a value or two of thousands
    assert _rel(got["out"], want["out"]) < 1e-5
    for a, b in zip(got["ins"], want["ins"]):
        assert _rel(a, b) < 2e-2
    for k in want["params"]:
        assert _rel(got["params"][k], want["params"][k]) < 2e-2, k


@pytest.mark.parametrize("which", [0, 1])
def test_layer_norm_modules_fused_chain(dev, which):
    """The bf16 chain against fp32, measured by torch's own autocast(bfloat16) run of the composition (which takes the
    layer-norm kernel on bf16 tensors)."""
    mod, call, ins, gout = list(_cases(dev, "layer"))[which]
    fp32 = _run(mod, call, ins, gout, fused=False)
    auto = _run(mod, call, ins, gout, fused=False, autocast=True)
    got = _run(mod, call, ins, gout, fused=True)
    assert got["out"].shape == fp32["out"].shape
    assert _rel(got["out"], fp32["out"]) < 1.6 * _rel(auto["out"], fp32["out"]) + 1e-3
    for a, c, b in zip(got["ins"], auto["ins"], fp32["ins"]):
        assert _rel(a, b) < 1.6 * _rel(c, b) + 1e-2
    for k in fp32["params"]:
        assert _rel(got["params"][k], fp32["params"][k]) < 1.6 * _rel(auto["params"][k], fp32["params"][k]) + 1e-2, k
    again = _run(mod, call, ins, gout, fused=True)
    assert torch.equal(got["out"], again["out"])


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("norm", ["batch", "layer"])
def test_inputs_kept_in_8_bits(dev, norm, which):
    """ACT_CKPT8: the same output; with BatchNorm the same input gradients and gradients of the norm's parameters; weight
    gradients within the 8-bit form's error; less memory held for the backward pass."""
    mod, call, ins, gout = list(_cases(dev, norm))[which]
    full = _run(mod, call, ins, gout, fused=True)
    kept = _run(mod, call, ins, gout, fused=True, ckpt8=True)
    assert torch.equal(full["out"], kept["out"])
    for k in full["params"]:
        if norm == "batch" and "conv" not in k:
            assert torch.equal(full["params"][k], kept["params"][k]), k
        else:
            # a value is off by at most 1/128 of its group's largest, which for these inputs is up to six times their rms
            assert _rel(kept["params"][k], full["params"][k]) < 6.0 / 128, k
    for a, b in zip(kept["ins"], full["ins"]):
        if norm == "batch":
            # (fp32 atomics in the weight gradients only; the gathers' backward adds in a fixed order)
            assert _rel(a, b) < 1e-6
        else:
            assert _rel(a, b) < 6.0 / 128
    assert kept["held"] < 0.85 * full["held"]
    again = _run(mod, call, ins, gout, fused=True, ckpt8=True)
    for k in kept["params"]:
        assert torch.equal(kept["params"][k], again["params"][k]), k              # no atomics left in the weight gradients


def test_network_with_layer_norm(dev):
    """The voting network with norm="layer": state_dict without buffers, a bf16 training step with and without kept 8-bit
    inputs (the same loss), an fp32 step, and an eval forward in which a cloud's features do not depend on the others."""
    from pvn3d_amd import train_step as ts
    from pvn3d_amd.lib.pointnet2_utils import _train_mlp
    torch.manual_seed(0)
    batch = ts.synthetic_batch(2, 4096, dev, seed_base=7, n_obj=1024)
    base = ts.PointVoteNet(norm="layer").to(dev)
    sd = base.backbone.state_dict()
    assert not list(base.backbone.buffers()) and any(k.endswith("normlayer.ln.weight") for k in sd)
    losses = {}
    for name, kw, flag in (("bf16", dict(autocast_dtype=torch.bfloat16), False), ("8 bits", dict(autocast_dtype=torch.bfloat16), True),
                           ("fp32", {}, False)):
        model = copy.deepcopy(base)
        opt = torch.optim.SGD(model.parameters(), lr=1e-3)
        _train_mlp.ACT_CKPT8 = flag
        try:
            losses[name] = float(ts.train_step(model, opt, batch, **kw))
        finally:
            _train_mlp.ACT_CKPT8 = False
        for n, p in model.named_parameters():
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
    assert losses["bf16"] == losses["8 bits"] and abs(losses["bf16"] - losses["fp32"]) < 2e-2 * abs(losses["fp32"])
    net = base.backbone.eval()
    with torch.no_grad():
        both, one = net(batch["pc"]), net(batch["pc"][:1].contiguous())
    assert _rel(both[:1], one) < 1e-5


def test_graphed_forward_with_layer_norm(dev):
    """The captured eval forward of a network with layer norm replays the eager one."""
    from pvn3d_amd.lib.pointnet2_msg import GraphedForward, Pointnet2MSG
    torch.manual_seed(0)
    net = Pointnet2MSG(norm="layer").to(dev).eval()
    clouds = _clouds(3, 4096, dev)
    pcs = [torch.cat([c, torch.rand(4096, 6, device=dev)], 1)[None].contiguous() for c in clouds]
    graphed = GraphedForward(net, pcs[0])
    for pc in pcs + pcs:
        got = graphed(pc).clone()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert _rel(got, net(pc)) < 1e-5


def test_unknown_norm_is_refused():
    from pvn3d_amd.lib.pointnet2_utils import pointnet2_modules as pm
    with pytest.raises(ValueError):
        pm.PointnetFPModule(mlp=[8, 8], norm="group")

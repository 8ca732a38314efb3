"""Which SharedMLPs the fused training chains take: their kernels read parameters by address, so those of another size, type
or device stay with torch, which converts or refuses them."""
import pytest
import torch
import torch.nn as nn

from pvn3d_amd.lib.layer_norm import LayerNorm
from pvn3d_amd.lib.pointnet2_utils import _train_mlp
from pvn3d_amd.lib.utils import pytorch_utils as pt_utils

CPU = torch.device("cpu")


def _mlp(norm, spec=(6, 8, 5)):
    return pt_utils.SharedMLP(list(spec), bn=norm == "batch", ln=norm == "layer").train()


def _norm(mlp, i, norm):
    seq = mlp[i].normlayer
    return (seq, "bn") if norm == "batch" else (seq, "ln")


@pytest.mark.parametrize("norm", ["batch", "layer"])
def test_parameters_the_kernels_cannot_read(norm):
    assert len(_train_mlp.shared_mlp_layers(_mlp(norm))) == 2 and len(_train_mlp.shared_mlp_layers(_mlp(norm), CPU)) == 2
    assert _train_mlp.shared_mlp_layers(_mlp(norm), torch.device("cuda", 0)) is None
    assert _train_mlp.shared_mlp_layers(_mlp(norm).bfloat16()) is None
    for c in (4, 16):                                                     # a norm of other channels than the layer's
        mlp = _mlp(norm)
        seq, name = _norm(mlp, 0, norm)
        setattr(seq, name, nn.BatchNorm2d(c) if norm == "batch" else LayerNorm(c, channel_dim=1))
        assert _train_mlp.shared_mlp_layers(mlp) is None
    mlp = _mlp(norm)                                                      # every second value of a longer tensor
    seq, name = _norm(mlp, 1, norm)
    getattr(seq, name).weight = nn.Parameter(torch.ones(10)[::2])
    assert _train_mlp.shared_mlp_layers(mlp) is None
    mlp = _mlp(norm)                                                      # layers that do not follow on each other
    mlp[1].conv = nn.Conv2d(9, 5, 1, bias=False)
    assert _train_mlp.shared_mlp_layers(mlp) is None


@pytest.mark.filterwarnings("ignore")
def test_weights_that_something_else_holds():
    """A weight norm replaces the parameter by an attribute of the same name: still the kernels' form."""
    mlp = _mlp("batch")
    nn.utils.weight_norm(mlp[0].conv)
    nn.utils.parametrizations.spectral_norm(mlp[1].conv)
    layers = _train_mlp.shared_mlp_layers(mlp)
    assert len(layers) == 2 and layers[0][0].weight.shape == (8, 6, 1, 1)


def test_no_running_statistics_to_update():
    """A BatchNorm whose buffers were taken away trains on the chain like one that has them."""
    mlp = _mlp("batch")
    for layer in mlp:
        layer.normlayer.bn.running_mean = layer.normlayer.bn.running_var = None
    assert len(_train_mlp.shared_mlp_layers(mlp)) == 2


@pytest.mark.parametrize("norm", ["batch", "layer"])
def test_inputs_of_other_channels(norm):
    """Features that a level was not built for are left to the composition (which refuses them)."""
    from pvn3d_amd.lib.pointnet2_utils import pointnet2_modules as pm
    sa = pm.PointnetSAModule([6, 8], npoint=4, radius=1.0, nsample=2, norm=norm).train()
    xyz, idx = torch.zeros(1, 9, 3), torch.zeros(1, 4, 2, dtype=torch.int32)
    for c in (5, 7):
        assert _train_mlp.sa_level_train(sa, xyz, xyz[:, :4], torch.zeros(1, c, 9), [idx]) is None
    assert _train_mlp.sa_level_train(sa, xyz, xyz[:, :4], None, [idx]) is None
    fp = pm.PointnetFPModule([6, 8], norm=norm).train()
    near = torch.zeros(1, 9, 3)
    for c in (1, 3):
        assert _train_mlp.fp_train(fp, torch.zeros(1, c, 9), torch.zeros(1, 4, 4), near.int(), near) is None

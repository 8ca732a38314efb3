"""What can be imported and used without the kernels' library."""
import os
import subprocess
import sys

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))

CODE = """
import torch
from pvn3d_amd.lib.utils import pytorch_utils as pt_utils
mlp = pt_utils.SharedMLP([6, 8, 5], bn=True)
assert mlp(torch.randn(2, 6, 3, 4)).shape == (2, 5, 3, 4)
try:
    pt_utils.SharedMLP([6, 8], ln=True)
except ImportError as e:
    assert "build it" in str(e)
else:
    raise AssertionError("a layer norm without its kernels")
"""


def test_shared_mlp_needs_only_torch(tmp_path):
    env = dict(os.environ, PVN3D_HIP_LIB=str(tmp_path / "none.so"))
    subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env=env, check=True, timeout=300)

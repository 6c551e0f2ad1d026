"""`networks` as a top-level package, as the reference has it (networks/networks.py): with genre-shapehd_amd/ on sys.path."""
import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "genre-shapehd_amd")


def run(code, **env):
    out = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, %r)\n" % PKG + code], capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, **env))
    assert out.returncode == 0 and "ok" in out.stdout, out.stderr[-2000:]


@pytest.mark.parametrize("env", ({}, {"GENRE_HIP_LIB": "/nonexistent/libgenre_hip.so"}), ids=("built", "without the native library"))
def test_networks_import_without_the_package(env):
    run("from networks.networks import ImageEncoder, Unet_3D, VoxelDecoder, VoxelGenerator, VoxelDiscriminator\n"
        "from networks.uresnet import Net, Net_inpaint\n"
        "import torch\n"
        "net = Unet_3D(nf=2)\n"
        "assert type(net.enc1.net[1]) is torch.nn.BatchNorm3d and VoxelDecoder(n_dims=8, nf=32)(torch.zeros(2, 8, 1, 1, 1)).shape[0] == 2\n"
        "print('ok')\n", **env)


def test_group_norm_is_found_there_too():
    run("from networks.networks import Unet_3D, VoxelGenerator\n"
        "from toolbox.group_norm.modules import GroupNormAct\n"
        "assert type(Unet_3D(nf=2, norm='group').enc1.net[1]) is GroupNormAct\n"
        "assert type(VoxelGenerator(nz=8, nf=4, norm='group').main[1]) is GroupNormAct\n"
        "print('ok')\n")

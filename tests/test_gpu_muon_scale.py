"""Matrices scaled to norm 1 without a step, up to the largest values there are."""
import pytest
import torch

from nerf_amd.muon_ops import newton_schulz

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("shape", [(2, 20, 30), (2, 60, 70), (2, 150, 300), (1, 700, 40), (2, 520, 600)], ids=str)
@pytest.mark.parametrize("scale", [1e-30, 1.0, 1e36, 3e38])
def test_no_step_at_all(shape, scale):
    """g / |g|: the scale 4096 / |g| and its product with g rounded, three half steps of fp32 with the result's (the power of two
    costs none)."""
    g = torch.rand(shape, generator=torch.Generator().manual_seed(1)) * 2 - 1
    g = (g.double() * scale).float()
    want = g.double() / g.double().square().sum((1, 2), keepdim=True).sqrt()
    got = newton_schulz(g.to(DEV), steps=0, eps=1e-30)
    assert ((got.double().cpu() - want).abs() <= 3 * 2.0 ** -24 * want.abs() + 2.0 ** -149).all()

"""The orthogonalised update at the ends of its sizes: as many matrices, a workgroup of 512 threads each, as a launch has no single
dimension for."""
import pytest
import torch

from nerf_amd import muon_ops
from nerf_amd.muon_ops import muon_update, newton_schulz

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
COUNT = (1 << 23) + 5
AT = [0, (1 << 22) - 1, 1 << 22, (1 << 23) - 1, 1 << 23, COUNT - 1]


def only_value():
    """what the iteration makes of a matrix' only singular value, 1"""
    a, b, c = muon_ops.COEFFICIENTS
    s = 1.0
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    return s


def test_more_matrices_than_a_grid_row():
    """Matrices of one row: each becomes its direction times the value above.  Every one of them is written: its norm is that
    value, off by half a step of fp16 per element (2^-11 of the norm in all; elements under fp16's smallest normal number, 2^-14,
    by 2^-25 each: 129^0.5 2^-25) and by the iteration's own fp32-class error, far under 2^-16."""
    g = torch.randn(COUNT, 1, 129, device=DEV, dtype=torch.float16, generator=torch.Generator(device=DEV).manual_seed(1))
    singly = [newton_schulz(g[at]) for at in AT]
    assert newton_schulz(g, out=g) is g
    for at, want in zip(AT, singly):
        assert torch.equal(g[at], want)
    s = only_value()
    for r in range(0, COUNT, 1 << 20):
        off = (g[r:r + (1 << 20)].float().square().sum((1, 2)).sqrt() - s).abs()
        assert float(off.max()) <= s * (2.0 ** -11 + 2.0 ** -16) + 129 ** 0.5 * 2.0 ** -25


def test_an_update_of_more_matrices_than_a_grid_row():
    gen = torch.Generator(device=DEV).manual_seed(2)
    p, g, m = (torch.randn(COUNT, 129, 1, device=DEV, generator=gen) for _ in range(3))
    singly = [[t[at].clone() for t in (p, g, m)] for at in AT]
    muon_update(p, g, m)
    for at, (p1, g1, m1) in zip(AT, singly):
        muon_update(p1, g1, m1)
        assert torch.equal(p[at], p1) and torch.equal(m[at], m1) and torch.equal(g[at], g1)

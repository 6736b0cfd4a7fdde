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


def test_overlapping_tensors_are_refused_and_neighbours_are_not():
    flat = torch.randn(3 * 600, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    first, second, third = flat.view(3, 2, 15, 20)
    want = newton_schulz(first)
    with pytest.raises(muon_ops.NrfError, match="overlaps"):
        newton_schulz(first, out=flat[300:900].view(2, 15, 20))
    assert torch.equal(newton_schulz(first, out=second), want) and torch.equal(second, want)
    start, grad = flat[300:900].clone().view(2, 15, 20), third.clone()
    for args in ((first, third, flat[300:900].view(2, 15, 20)), (flat[300:900].view(2, 15, 20), first, third),
                 ([first, flat[1:601].view(2, 15, 20)], [third, third], [torch.zeros_like(first), torch.zeros_like(first)])):
        with pytest.raises(muon_ops.NrfError, match="overlap"):
            muon_update(*args)
    assert torch.equal(flat[300:900].view(2, 15, 20), start) and torch.equal(third, grad)
    p, m = first.clone(), second.clone()
    muon_update(p, third, m)
    muon_update(first, third, second)                        # neighbours of one buffer
    assert torch.equal(first, p) and torch.equal(second, m) and torch.equal(third, grad)
    # a transposed gradient is laid out anew before the call
    square = torch.randn(8, 8, device=DEV)
    p, m = square.clone(), torch.zeros_like(square)
    muon_update(p, square.t().contiguous(), m)
    q = square.clone()
    muon_update(q, q.t(), torch.zeros_like(q))
    assert torch.equal(p, q)


def test_a_list_of_more_matrices_than_one_call_takes():
    """3 x 22000 matrices of 1 x 545, of which a call takes 65535: each tensor alone would be taken"""
    gen = torch.Generator(device=DEV).manual_seed(4)
    p, g, m = ([torch.randn(22000, 1, 545, device=DEV, generator=gen) for _ in range(3)] for _ in range(3))
    singly = [[t.clone() for t in ts] for ts in zip(p, g, m)]
    muon_update(p, g, m)
    for i, (p1, g1, m1) in enumerate(singly):     # (whole tensors: a few matrices alone take the launch-per-step kernel)
        muon_update(p1, g1, m1)
        assert torch.equal(p[i], p1) and torch.equal(m[i], m1)
    with pytest.raises(muon_ops.NrfError, match="up to 65535"):
        muon_update(*([torch.zeros(65536, 1, 545, device=DEV) for _ in range(2)] for _ in range(3)))

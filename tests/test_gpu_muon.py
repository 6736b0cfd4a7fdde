"""The orthogonalised update (nerf_amd/muon_ops.py) against its definition in 64 bits, by singular values: with G = U s V^T the
result is U f(f(..f(s / |s|))) V^T, f(s) = a s + b s^3 + c s^5.

Tolerances.  The products' operands are rounded to 2^-22 where an iteration in fp32 rounds to 2^-24, the sums are fp32 in both:
a result may be off by 4 times what the same iteration in fp32 on the CPU is off for the same input, in the 2-norm over the
matrix, and by 4 2^-22 of the result where that one is exact by chance.  The output's own rounding adds half a step.

The terms end at fp16's smallest step 2^-24: at the scale 2^12 an entry of X is held to 2^-37 whatever its size (half a step).
That error grows by at most the iteration's steepest slope, a, in every step that follows: over a matrix of m x n entries it
adds 2^-37 sqrt(m n) (a + a^2 + ... + a^steps), 2e-7 for 32 x 40 and five steps.  It shows only where the whole matrix is
that small, norms far under eps (measured before this term was written: 7.6e-8 at a norm of 1e-8 eps)."""
import numpy as np
import pytest
import torch

from nerf_amd import muon_ops
from nerf_amd.muon_ops import muon_update, newton_schulz

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ABC = muon_ops.COEFFICIENTS


def definition(g, steps=5, abc=ABC, eps=1e-7):
    u, s, vh = torch.linalg.svd(g.double().cpu(), full_matrices=False)
    s = s / s.square().sum(-1, keepdim=True).sqrt().clamp(min=eps)
    for _ in range(steps):
        s = abc[0] * s + abc[1] * s ** 3 + abc[2] * s ** 5
    return (u * s[..., None, :]) @ vh


def iteration32(g, steps=5, abc=ABC, eps=1e-7):
    x = g.float().cpu()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / x.double().square().sum((-1, -2), keepdim=True).sqrt().clamp(min=eps).float()
    for _ in range(steps):
        A = x @ x.transpose(-1, -2)
        x = abc[0] * x + (abc[1] * A + abc[2] * A @ A) @ x
    return x.transpose(-1, -2) if tall else x


def norm(x):
    return x.double().square().sum((-1, -2)).sqrt()


def bound(g, want, dtype, **kw):
    off32 = norm(iteration32(g, **kw).double() - want)
    a = max(1.0, kw.get("abc", ABC)[0])
    floor = 2.0 ** -37 * (g.shape[-1] * g.shape[-2]) ** 0.5 * sum(a ** k for k in range(1, kw.get("steps", 5) + 1))
    return floor + 4 * off32 + 4 * 2.0 ** -22 * norm(want) + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2.0 ** -24) * norm(want)


def gradient(batch, m, n, seed=0, dtype=torch.float32, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 8)
    x = torch.randn(batch, m, n, generator=g) + torch.randn(batch, m, r, generator=g) @ torch.randn(batch, r, n, generator=g) / r ** 0.5
    return (scale * x).to(dtype)


SHAPES = [(1, 1, 1), (3, 1, 7), (2, 7, 1), (5, 2, 2), (4, 31, 33), (9, 32, 32), (7, 32, 63), (6, 63, 32), (5, 32, 64), (3, 20, 128),
          (3, 128, 32), (2, 17, 100), (1, 32, 129), (2, 33, 33), (2, 40, 7), (2, 64, 64), (2, 65, 130), (1, 130, 65), (3, 64, 544), (2, 545, 64), (1, 544, 33), (2, 33, 48), (3, 128, 160), (2, 160, 127), (1, 161, 128), (2, 97, 97), (1, 1, 544),
          (2, 500, 1), (1, 129, 129), (2, 96, 112), (3, 100, 640), (2, 640, 101), (1, 64, 576), (5, 33, 601), (2, 641, 70), (1, 128, 192),
          (40, 128, 165), (90, 120, 190), (17, 10, 600), (2, 128, 283),
          (1, 283, 128), (3, 256, 256), (1, 513, 600), (1, 600, 514), (1, 5, 700), (300, 16, 16)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_newton_schulz(shape, dtype):
    g = gradient(*shape, seed=sum(shape), dtype=DT[dtype], scale=1.0 if dtype == "fp16" else 1e-3)
    got = newton_schulz(g.to(DEV))
    want = definition(g)
    assert got.dtype == DT[dtype] and got.shape == g.shape
    off, most = norm(got.double().cpu() - want), bound(g, want, DT[dtype])
    assert (off <= most).all(), (off / most).max()
    assert torch.equal(got, newton_schulz(g.to(DEV)))                     # the same bits on every run


@pytest.mark.parametrize("shape", [(2, 32, 48), (2, 70, 96)], ids=str)
@pytest.mark.parametrize("steps,abc", [(0, ABC), (1, ABC), (2, ABC), (10, (1.5, -0.5, 0.0)), (8, (2.0, -1.5, 0.5))])
def test_steps_and_coefficients(shape, steps, abc):
    g = gradient(*shape, seed=steps)
    got = newton_schulz(g.to(DEV), steps=steps, coefficients=abc)
    want = definition(g, steps, abc)
    assert (norm(got.double().cpu() - want) <= bound(g, want, torch.float32, steps=steps, abc=abc)).all()


@pytest.mark.parametrize("shape", [(3, 32, 40), (3, 96, 80)], ids=str)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e18, 1e36])
def test_magnitudes(shape, scale):
    """The result does not depend on the scale, up to the smallest norm, whose matrices shrink with it; no sum overflows."""
    g = gradient(*shape, seed=1, scale=1.0) * scale
    got = newton_schulz(g.to(DEV), eps=1e-20)
    want = definition(g, eps=1e-20)
    assert (norm(got.double().cpu() - want) <= bound(g, want, torch.float32, eps=1e-20)).all()


@pytest.mark.parametrize("shape", [(4, 32, 40), (4, 40, 31), (4, 96, 80), (4, 64, 200)], ids=str)
def test_zero_low_rank_and_not_finite_matrices(shape):
    g = gradient(*shape, seed=2)
    clean = newton_schulz(g.to(DEV))
    g[1] = 0
    g[2, 3, 4] = float("nan")
    got = newton_schulz(g.to(DEV))
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])          # the others of the batch
    assert (got[1] == 0).all() and torch.isnan(got[2]).all()
    g[2] = torch.outer(torch.arange(1.0, shape[1] + 1), torch.linspace(-1, 1, shape[2]))     # rank one: one singular value, 1
    got, want = newton_schulz(g.to(DEV)), definition(g)
    assert norm(got[2].double().cpu() - want[2]) <= bound(g[2:3], want[2:3], torch.float32)[0]
    g[2, 0, 0] = float("inf")
    assert torch.isnan(newton_schulz(g.to(DEV))[2]).all()


@pytest.mark.parametrize("shape", [(3, 20, 24), (3, 100, 31), (3, 60, 70), (3, 100, 140), (3, 150, 90), (3, 200, 130), (3, 64, 2000)], ids=str)
@pytest.mark.parametrize("steps", [0, 5])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_one_bad_value_is_nan_everywhere_in_its_matrix_alone(shape, steps, bad):
    g = gradient(*shape).to(DEV)
    clean = newton_schulz(g, steps=steps)
    g[1, 7, 11] = bad
    got = newton_schulz(g, steps=steps)
    assert got[1].isnan().all() and torch.equal(got[[0, 2]], clean[[0, 2]])
    p, m = torch.zeros_like(g), torch.zeros_like(g)
    clipped = newton_schulz(g.clamp(-40, 40), steps=steps)       # an infinite gradient is clipped, NaN stays
    muon_update(p, g, m, lr=1.0, momentum=0.0, steps=steps)
    scale = max(1.0, shape[1] / shape[2]) ** 0.5
    assert bool(p[1].isnan().all()) == (bad != bad)
    off = (p + scale * clipped)[[0, 2] if bad != bad else [0, 1, 2]].abs()
    assert float(off.max()) <= 4 * 2.0 ** -24 * scale * float(clipped.nan_to_num().abs().max())     # the rate and the product rounded


def test_views_and_in_place():
    g = gradient(3, 48, 80, seed=3).to(DEV)
    want = newton_schulz(g)
    assert torch.equal(newton_schulz(g.transpose(1, 2).contiguous().transpose(1, 2)), want)
    odd = torch.zeros(g.numel() + 1, device=DEV)[1:].view_as(g)
    odd.copy_(g)
    assert torch.equal(newton_schulz(odd), want)
    assert torch.equal(newton_schulz(g[1]), want[1])                                 # one matrix
    assert newton_schulz(odd, out=odd) is odd and torch.equal(odd, want)
    small = gradient(5, 20, 30, seed=4).to(DEV)
    want = newton_schulz(small)
    assert torch.equal(newton_schulz(small, out=small), want)
    assert newton_schulz(torch.zeros(0, 8, 8, device=DEV)).shape == (0, 8, 8)


def test_wide_and_tall_are_each_others_transpose():
    for shape in ((4, 24, 90), (2, 70, 150)):
        g = gradient(*shape, seed=5)
        a = newton_schulz(g.to(DEV)).cpu()
        b = newton_schulz(g.transpose(1, 2).contiguous().to(DEV)).transpose(1, 2).cpu()
        want = definition(g)
        assert (norm(a.double() - b.double()) <= 2 * bound(g, want, torch.float32)).all()


def muon64(p, g, m, lr, mu, nesterov, wd, clip, scale, dtype=torch.float64):
    g = (g.to(dtype) * scale).clamp(-clip, clip)
    m = mu * m.to(dtype) + g
    u = g + mu * m if nesterov else m
    o = definition(u) if dtype == torch.float64 else iteration32(u)
    return (1 - lr * wd) * p.to(dtype) - lr * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5 * o, m, o


@pytest.mark.parametrize("shape", [(5, 32, 63), (3, 63, 32), (2, 128, 283), (2, 283, 128), (1, 256, 256), (4, 3, 128), (2, 600, 520), (3, 64, 300), (2, 150, 110), (3, 62, 620), (4, 333, 99)], ids=str)
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(shape, nesterov):
    gen = torch.Generator().manual_seed(7)
    p, m = torch.randn(shape, generator=gen) / shape[2] ** 0.5, 2e-3 * torch.randn(shape, generator=gen)
    pd, md = p.to(DEV), m.to(DEV)
    opt = dict(lr=0.1, weight_decay=0.3, clip_value=2e-3, grad_scale=0.5)
    p64, m64 = p, m
    for step in range(2):
        g = gradient(*shape, seed=10 + step)
        gd = g.to(DEV)
        start_p, start_m = pd.cpu(), md.cpu()
        version = pd._version
        muon_update(pd, gd, md, momentum=0.9, nesterov=nesterov, **opt)
        assert pd._version > version and torch.equal(gd.cpu(), g)
        p64, m64, o = muon64(start_p, g, start_m, 0.1, 0.9, nesterov, 0.3, 2e-3, 0.5)
        _, _, o32 = muon64(start_p, g, start_m, 0.1, 0.9, nesterov, 0.3, 2e-3, 0.5, torch.float32)
        # half a step each: the result, mu (0.9 is not an fp32 number) times the old momentum, and g, which is at most the clip
        # value 2e-3 (itself not an fp32 number)
        assert ((md.double().cpu() - m64).abs() <= 2.0 ** -24 * (m64.abs() + 2 * start_m.double().abs() + 2e-3)).all()
        rate = 0.1 * max(1.0, shape[1] / shape[2]) ** 0.5
        # O as above; decay, rate, their products and the sum: five half steps of the terms
        off = rate * (4 * norm(o32.double() - o) + 4 * 2.0 ** -22 * norm(o)) + 5 * 2.0 ** -24 * (norm(p64) + rate * norm(o))
        assert (norm(pd.double().cpu() - p64) <= off).all()


@pytest.mark.parametrize("shape,count", [((40, 24), 3), ((2, 100, 90), 2), ((6, 5), 40)], ids=str)
def test_muon_on_a_list_of_tensors(shape, count):
    """Tensors at odd places of one buffer, more of them than one call takes: the bits of one call each."""
    gen = torch.Generator().manual_seed(8)
    numel = int(np.prod(shape))
    flat = torch.randn(3, count, numel + 1, generator=gen).to(DEV)
    views = [[row[1:].view(shape) for row in part] for part in flat]
    singly = [[t.clone() for t in ts] for ts in views]
    muon_update(*views, lr=0.05)
    for p, g, m in zip(*singly):
        muon_update(p, g, m, lr=0.05)
    for got, want in zip(views, singly):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(flat[:, :, 0].cpu(), torch.randn(3, count, numel + 1, generator=torch.Generator().manual_seed(8))[:, :, 0])


@pytest.mark.parametrize("shape", [(50, 32, 63), (3, 100, 120), (2, 128, 283)], ids=str)
def test_muon_on_a_side_stream_and_in_a_graph(shape):
    p0, g0 = gradient(*shape, seed=1).to(DEV), gradient(*shape, seed=2).to(DEV)

    def steps(p, m, count):
        for _ in range(count):
            muon_update(p, g0, m)

    want_p, want_m = p0.clone(), torch.zeros_like(p0)
    steps(want_p, want_m, 3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        p, m = p0.clone(), torch.zeros_like(p0)
        steps(p, m, 3)
    side.synchronize()
    assert torch.equal(p, want_p) and torch.equal(m, want_m)
    p, m = p0.clone(), torch.zeros_like(p0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_update(p, g0, m)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        steps(p0.clone(), torch.zeros_like(p0), 1)             # eager work between the replays
    torch.cuda.synchronize()
    assert torch.equal(p, want_p) and torch.equal(m, want_m)


@pytest.mark.parametrize("shape", [(1, 256, 8192), (3, 64, 4096), (2, 1000, 70), (1, 4500, 129), (1, 640, 1152), (1, 33, 40000)], ids=str)
def test_long_sums_are_split(shape):
    """few tiles and a long k: A = X X^T from parts"""
    g = gradient(*shape, seed=sum(shape))
    got, want = newton_schulz(g.to(DEV)), definition(g)
    off, most = norm(got.double().cpu() - want), bound(g, want, torch.float32)
    assert (off <= most).all(), (off / most).max()
    assert torch.equal(got, newton_schulz(g.to(DEV)))


@pytest.mark.parametrize("batch,m,n", [(100003, 3, 5), (70001, 34, 33), (66000, 20, 60)])
def test_many_matrices(batch, m, n):
    g = torch.randn(batch, m, n, generator=torch.Generator(device=DEV).manual_seed(batch), device=DEV)
    got = newton_schulz(g)
    for at in (0, 65535, 65536, batch - 1):
        assert torch.equal(got[at], newton_schulz(g[at]))
    pick = torch.tensor([1, 65534, 65537, batch - 2])
    want = definition(g[pick.to(DEV)])
    assert (norm(got[pick.to(DEV)].double().cpu() - want) <= bound(g[pick.to(DEV)], want, torch.float32)).all()


def test_planes_of_more_than_2_gib():
    """One non-zero per row, in columns of their own: every singular value goes its own way, x -> a x + b x^3 + c x^5.  A plane of
    X takes 2.2 GiB, both 4.3: offsets past 32 bits.  Off by the output's rounding and the floor of the terms (no sums: each
    has one addend)."""
    m, n = 16450, 65500
    at = (torch.arange(m) * 65123 + 77) % n
    assert at.unique().numel() == m
    s = torch.rand(m, generator=torch.Generator().manual_seed(1)) + 0.5
    g = torch.zeros(m, n, dtype=torch.bfloat16, device=DEV)
    rows = torch.arange(m, device=DEV)
    g[rows, at.to(DEV)] = s.bfloat16().to(DEV)
    x = s.bfloat16().double()
    x = x / x.square().sum().sqrt()
    want = ABC[0] * x + ABC[1] * x ** 3 + ABC[2] * x ** 5
    newton_schulz(g, steps=1, out=g)
    got = g[rows, at.to(DEV)].double().cpu()
    assert ((got - want).abs() <= 2.0 ** -8 * want + 2.0 ** -20 * want + 4 * 2.0 ** -37).all()
    g[rows, at.to(DEV)] = 0
    assert not bool(g.any())


def test_refusals():
    E = muon_ops.NrfError
    g = torch.zeros(2, 8, 8, device=DEV)
    for bad in (g.cpu(), g.double(), g.int(), g[0, 0], g[None]):
        with pytest.raises(E):
            newton_schulz(bad)
    for kw in (dict(steps=17), dict(steps=-1), dict(eps=0.0), dict(coefficients=(4.0, 0.0, 0.0)), dict(coefficients=(3.4445, 4.775, 2.0)),
               dict(out=g.bfloat16()), dict(out=torch.zeros(2, 8, 7, device=DEV)), dict(out=g.transpose(1, 2))):
        with pytest.raises(E):
            newton_schulz(g, **kw)
    for args in ((g, g[0], g), (g, g.bfloat16(), g), (g.cpu(), g, g), (g.transpose(1, 2), g, g), ([g], [g, g], [g]), (g[0, 0], g[0, 0], g[0, 0])):
        with pytest.raises(E):
            muon_update(*args)
    h, k = torch.zeros_like(g), torch.zeros_like(g)
    for args in ((g, h, g), (g, g, h), (g, h, h), ([g, g], [h, h], [k, k.clone()]), ([g, k], [h, h], [k, h.clone()])):
        with pytest.raises(E):
            muon_update(*args)
    for kw in (dict(clip_value=0.0), dict(momentum=1.0), dict(steps=99)):
        with pytest.raises(E):
            muon_update(g, g.clone(), g.clone(), **kw)
    assert muon_update([], [], []) is None

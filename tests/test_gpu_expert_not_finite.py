"""Operands that are not finite: every output whose sum holds one is not finite, every other has the bits that it has without."""
import pytest
import torch

from nerf_amd.expert_ops import expert_linear, expert_linear_backward, expert_plan

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
N, E = 300, 4
INF, NAN = float("inf"), float("nan")
# fp32: the two forms of the arithmetic and odd sizes of the first's 32 x 32 blocks; 16-bit: the general tile and the wide one
LAYERS = [(63, 32, "fp32"), (32, 20, "fp32"), (64, 64, "fp32"), (40, 33, "fp32"), (5, 3, "fp32"), (65, 64, "fp32"), (200, 70, "fp32"),
          (63, 32, "bf16"), (136, 128, "bf16"), (65, 40, "fp16"), (256, 136, "fp16")]


def layer(k, m, dtype):
    g = torch.Generator().manual_seed(k + m)
    dtype = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    x, w, b, dy = (torch.randn(s, generator=g).to(dtype).to(DEV) for s in ((N, k), (E, m, k), (E, m), (N, m)))
    return x, w / 8, b, dy, torch.randint(-1, E, (N,), generator=g, dtype=torch.int32).to(DEV)


def check(got, clean, reached, name):
    assert not got[reached].isfinite().any(), name
    assert torch.equal(got[~reached], clean[~reached]), name


@pytest.mark.parametrize("k,m,dtype", LAYERS)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_forward(k, m, dtype, bad):
    x, w, b, _, index = layer(k, m, dtype)
    plan = expert_plan(index, E)
    clean = expert_linear(x, w, b, plan)
    rows = [int((index == e).nonzero()[i, 0]) for e, i in ((0, 0), (1, 3), (3, -1))]
    reached = torch.zeros(N, m, dtype=torch.bool, device=DEV)
    x[rows[0], 0], x[rows[1], k - 1], x[rows[2], k // 2] = bad, bad, bad
    reached[rows] = True
    w[2, m - 1, k - 1], w[2, 0, 0] = bad, bad
    b[2, m // 2] = bad
    for feature in (0, m // 2, m - 1):
        reached[index == 2, feature] = True
    check(expert_linear(x, w, b, plan), clean, reached, "y")


@pytest.mark.parametrize("k,m,dtype", LAYERS)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_backward(k, m, dtype, bad):
    x, w, _, dy, index = layer(k, m, dtype)
    plan = expert_plan(index, E)
    clean = expert_linear_backward(dy, x, w, plan)
    rows = [int((index == e).nonzero()[i, 0]) for e, i in ((0, 0), (1, 3), (3, -1))]
    dx, dw, db = (torch.zeros(t.shape, dtype=torch.bool, device=DEV) for t in clean)
    x[rows[0], k - 1] = bad
    dw[0, :, k - 1] = True
    w[2, m - 1, 0] = bad
    dx[index == 2, 0] = True
    for r, e, feature in ((rows[1], 1, m - 1), (rows[2], 3, 0)):
        dy[r, feature] = bad
        dx[r], dw[e, feature], db[e, feature] = True, True, True
    none = int((index == -1).nonzero()[0, 0])
    x[none], dy[none] = bad, bad                        # of no expert: reaches nothing
    for name, got, was, reached in zip(("x", "weight", "bias"), expert_linear_backward(dy, x, w, plan), clean, (dx, dw, db)):
        check(got, was, reached, name)


def test_the_two_forms_of_fp32():
    """An infinite input of a layer of 64 stays infinite, of 65 it gives NaN; where infinities cancel both give NaN."""
    for k, stays in ((64, True), (65, False)):
        x, w, b, _, index = layer(k, 8, "fp32")
        index[:2] = 0
        w[0] = w[0].abs() + 0.1
        x[0, 3], x[1, 3], x[1, 4] = INF, INF, -INF
        y = expert_linear(x, w, b, expert_plan(index, E))
        assert bool((y[0] == INF).all()) == stays and bool(y[0].isnan().all()) != stays
        assert y[1].isnan().all()

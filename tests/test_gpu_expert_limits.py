"""The expert products at the ends of their sizes: as many workgroups as a launch has no single dimension for."""
import pytest
import torch

from nerf_amd.expert_ops import expert_linear, expert_linear_backward, expert_plan

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E, WIDTH = 16384, 65536     # tiles of 64 outputs: 2^24 workgroups of 256 threads, 2^32 work-items


def pairs(n, seed):
    """n rows over all experts (the first E one each), weights of one input: every output is one product"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, 1, device=DEV, generator=g).bfloat16()
    w = torch.randn(E, WIDTH, 1, device=DEV, generator=g, dtype=torch.bfloat16)
    index = torch.cat([torch.randperm(E, device=DEV, generator=g), torch.full((max(0, n - E),), -1, device=DEV)])[:n].to(torch.int32)
    return x, w, index


def test_every_expert_with_the_widest_layer():
    """A product of two bf16 values is exact in fp32, so the outputs and the weights' gradients are equal to the bit.  dx adds
    65536 of them: k 2^-23 of the magnitudes' sum and half a step, as for every 16-bit product."""
    n = E + 9
    x, w, index = pairs(n, 1)
    plan = expert_plan(index, E)
    y = expert_linear(x, w, None, plan)
    for r in range(0, E, 2048):
        at = index[r:r + 2048].long()
        assert torch.equal(y[r:r + 2048], (x[r:r + 2048].float() * w[at, :, 0].float()).bfloat16())
    assert not y[E:].any()
    dy = y                                       # any gradient will do
    dx, dw, db = expert_linear_backward(dy, x, w, plan)
    for r in range(0, E, 2048):
        at = index[r:r + 2048].long()
        assert torch.equal(dw[at, :, 0], (dy[r:r + 2048].float() * x[r:r + 2048].float()).bfloat16())
        assert torch.equal(db[at], dy[r:r + 2048])
    assert not dx[E:].any()
    for r in (0, 1, 777, E - 1):
        product = dy[r].double() * w[int(index[r]), :, 0].double()
        want, size = float(product.sum()), float(product.abs().sum())
        assert abs(float(dx[r, 0]) - want) <= WIDTH * 2.0 ** -23 * size + 2.0 ** -8 * abs(want)


@pytest.mark.parametrize("n", [1, 3])
def test_a_few_tokens_through_the_widest_layer(n):
    x, w, index = pairs(n, 2)
    y = expert_linear(x, w, None, expert_plan(index, E))
    assert torch.equal(y, (x.float() * w[index.long(), :, 0].float()).bfloat16())


def test_as_many_rows_as_there_may_be():
    """2^28 rows through layers of 1 -> 1 in fp32.  Inputs of +-1 and gradients of 1: every sum is a whole number, the result off by
    half a step of fp32; outputs are the weights or their negatives."""
    n, count = 1 << 28, 5
    g = torch.Generator(device=DEV).manual_seed(3)
    index = torch.randint(-1, count, (n,), device=DEV, generator=g, dtype=torch.int32)
    index[-1] = count - 1
    plan = expert_plan(index, count)
    counts = torch.stack([(index == e).sum() for e in range(count)])
    assert torch.equal(plan.counts.long(), counts) and plan.offsets.tolist() == [0] + torch.cumsum(counts, 0).tolist()
    key = torch.where(index < 0, count, index)[plan.order.long()]
    assert bool((key[1:] >= key[:-1]).all()) and bool(((plan.order[1:] > plan.order[:-1]) | (key[1:] > key[:-1])).all())
    del key
    x = (torch.randint(0, 2, (n, 1), device=DEV, generator=g, dtype=torch.int8) * 2 - 1).float()
    w = torch.randn(count, 1, 1, device=DEV, generator=g)
    table = torch.cat([w.flatten(), torch.zeros(1, device=DEV)])
    y = expert_linear(x, w, None, plan)
    for r in range(0, n, 1 << 26):
        at = index[r:r + (1 << 26)].long()
        assert torch.equal(y[r:r + (1 << 26), 0], table[at] * x[r:r + (1 << 26), 0])
    dx, dw, db = expert_linear_backward(torch.ones_like(x), x, w, plan)
    for e in range(count):
        rows = index == e
        want = int(x[:, 0][rows].sum(dtype=torch.float64))
        assert abs(float(dw[e, 0, 0]) - want) <= 2.0 ** -24 * abs(want) and abs(float(db[e, 0]) - int(counts[e])) <= 2.0 ** -24 * int(counts[e])
        assert bool((dx[:, 0][rows] == w[e, 0, 0]).all())
    assert not bool(dx[:, 0][index < 0].any())


def test_as_many_rows_and_experts():
    """the plan alone, every key in use"""
    n = 1 << 28
    index = torch.arange(n, device=DEV, dtype=torch.int32) * 7 % (E + 1)        # E: of no expert
    plan = expert_plan(index, E)
    counts = torch.bincount(index, minlength=E + 1)
    assert torch.equal(plan.counts.long(), counts[:E]) and torch.equal(plan.offsets.long(), torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(counts[:E], 0)]))
    key = index[plan.order.long()]
    assert bool((key[1:] >= key[:-1]).all()) and bool(((plan.order[1:] > plan.order[:-1]) | (key[1:] > key[:-1])).all())

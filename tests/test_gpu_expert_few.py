"""Few experts with many rows each: the sums of dW and db over an expert's parts, dealt to wavefronts from 32 parts on."""
import pytest
import torch

from nerf_amd.expert_ops import expert_linear_backward, expert_plan

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("rows", [[8191], [8192], [8193], [30000, 257, 0, 256, 7936, 7937], [31 * 256, 1, 100000]], ids=str)
@pytest.mark.parametrize("n_in,n_out", [(64, 64), (3, 2), (1, 1), (80, 81), (33, 17)])
def test_whole_numbers(rows, n_in, n_out):
    """Small whole numbers: every product and every sum is exact (under 2^24), whatever the order, so the result is too."""
    g = torch.Generator().manual_seed(len(rows) + n_in)
    index = torch.cat([torch.full((r,), e) for e, r in enumerate(rows)])
    index = index[torch.randperm(len(index), generator=g)]
    x, dy = (torch.randint(-3, 4, (len(index), k), generator=g).float() for k in (n_in, n_out))
    w = torch.zeros(len(rows), n_out, n_in)
    plan = expert_plan(index.to(torch.int32).to(DEV), len(rows))
    _, dw, db = expert_linear_backward(dy.to(DEV), x.to(DEV), w.to(DEV), plan, want_x=False)
    for e in range(len(rows)):
        part = dy[index == e].double()
        assert torch.equal(dw[e].double().cpu(), part.T @ x[index == e].double())
        assert torch.equal(db[e].double().cpu(), part.sum(0))

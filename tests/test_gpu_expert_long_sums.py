"""dW and db over very many rows, whose parts of 256 rows are added one after the other."""
import pytest
import torch

from nerf_amd.expert_ops import expert_linear_backward, expert_plan

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("n,n_in,n_out,extra", [((1 << 26) + 77, 1, 1, 15 / 2048), ((1 << 24) + 300, 65, 2, 7 / 4096)])
def test_equal_rows(n, n_in, n_out, extra):
    """Rows of ones with gradients of 1 + extra: the products and the sums of a run (at most 257, 12 bits behind the point) are exact
    in fp32, so the result is off by its own rounding alone, half a step.  A part's `extra` lies under half a step of the whole
    sum's second half: a running sum in 32 bits is 0.4 % and 0.09 % off."""
    x = torch.ones(n, n_in, device=DEV)
    dy = torch.full((n, n_out), 1 + extra, device=DEV)
    w = torch.ones(2, n_out, n_in, device=DEV)
    index = torch.ones(n, dtype=torch.int32, device=DEV)
    index[:300] = 0
    index[-50:] = -1
    _, dw, db = expert_linear_backward(dy, x, w, expert_plan(index, 2), want_x=False)
    for e, rows in ((0, 300), (1, n - 350)):
        want = rows * (1 + extra)
        assert float((dw[e].double() - want).abs().max()) <= 2.0 ** -24 * want
        assert float((db[e].double() - want).abs().max()) <= 2.0 ** -24 * want


@pytest.mark.parametrize("n,n_in,n_out,dtype", [(6000011, 64, 5, "fp32"), (2000003, 70, 40, "fp32"), (3000001, 264, 136, "bf16"),
                                                (3000001, 264, 136, "fp16"), (2000003, 100, 9, "fp16")])
def test_random_rows(n, n_in, n_out, dtype):
    """By norm.  Products of independent normal values: a sum over r rows is some sqrt(r) in size.  An addition inside a run of 256
    rows rounds by 2^-24 of a sum of about 16, and the errors of n additions add like the products do, as a root: 2^-20 of the
    result in all, three bf16 terms per operand leave out less.  The longer chains of the 16-bit kernels (64 shares of an
    expert's rows at most: sums of sqrt(r / 64)) stay under 2^-15.  Then half a step of the output's type; twice that here."""
    g = torch.Generator(device=DEV).manual_seed(n_in)
    x, dy = (torch.randn(n, k, device=DEV, generator=g).to(DT[dtype]) for k in (n_in, n_out))
    w = torch.zeros(3, n_out, n_in, device=DEV, dtype=DT[dtype])
    index = torch.randint(-1, 3, (n,), device=DEV, generator=g, dtype=torch.int32)
    _, dw, db = expert_linear_backward(dy, x, w, expert_plan(index, 3), want_x=False)
    most = 2 * (2.0 ** -20 if dtype == "fp32" else 2.0 ** -15 + torch.finfo(DT[dtype]).eps / 2)
    for e in range(3):
        want, bias = torch.zeros(n_out, n_in, dtype=torch.float64, device=DEV), torch.zeros(n_out, dtype=torch.float64, device=DEV)
        for r in range(0, n, 1 << 20):
            part = dy[r:r + (1 << 20)].double() * (index[r:r + (1 << 20)] == e)[:, None]
            want += part.T.contiguous() @ x[r:r + (1 << 20)].double()
            bias += part.sum(0)
        assert float((dw[e].double() - want).norm() / want.norm()) <= most
        assert float((db[e].double() - bias).norm() / bias.norm()) <= most

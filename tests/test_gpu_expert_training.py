"""The expert operators and the Muon update as a program uses them together: rows grouped by expert, two layers forward and
backward, the weights updated, all of it again.

Each operator is held against its definition in 64 bits on the operands that it was given, the outputs of the one before.
Tolerances.  fp32 products are three bf16 terms per operand: (6 k + 3) 2^-23 of the sum of the products' magnitudes over k
products, and half a step of the result.  bf16 and fp16 products are exact, k 2^-23 and half a step.  The update: four times
what the same iteration in fp32 on the CPU is off, and four times 2^-22 of the step; then the sum's own half step."""
import pytest
import torch

from nerf_amd.expert_ops import expert_linear, expert_linear_backward, expert_plan
from nerf_amd.muon_ops import COEFFICIENTS as ABC
from nerf_amd.muon_ops import muon_update, newton_schulz

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def near(got, want, magnitude, k):
    per = 6 * k + 3 if got.dtype == torch.float32 else k
    info = torch.finfo(got.dtype)
    most = per * 2.0 ** -23 * magnitude + info.eps / 2 * (want.abs() + info.tiny)
    off = (got.double().cpu() - want).abs()
    assert (off <= most).all(), (off / most).max()


def chosen(index, E):
    return [(index == e).nonzero()[:, 0] for e in range(E)]


def check_layer(x, w, b, y, index, relu):
    x, w, b, index = x.double().cpu(), w.double().cpu(), b.double().cpu(), index.cpu().long()
    want, size = torch.zeros(len(x), w.shape[1], dtype=torch.float64), torch.zeros(len(x), w.shape[1], dtype=torch.float64)
    for e, rows in enumerate(chosen(index, len(w))):
        want[rows], size[rows] = x[rows] @ w[e].T + b[e], x[rows].abs() @ w[e].abs().T + b[e].abs()
    near(y, want.clamp(min=0) if relu else want, size, x.shape[1] + 1)


def check_gradients(dy, x, w, y, index, dx, dw, db):
    dz = (dy.double() * (y.double() > 0) if y is not None else dy.double()).cpu()
    x, w, index = x.double().cpu(), w.double().cpu(), index.cpu().long()
    want, size = torch.zeros_like(x), torch.zeros_like(x)
    for e, rows in enumerate(chosen(index, len(w))):
        want[rows], size[rows] = dz[rows] @ w[e], dz[rows].abs() @ w[e].abs()
        near(dw[e], dz[rows].T @ x[rows], dz[rows].T.abs() @ x[rows].abs(), max(1, len(rows)))
        near(db[e], dz[rows].sum(0), dz[rows].abs().sum(0), max(1, len(rows)))
    near(dx, want, size, w.shape[1])


def iteration(u):
    tall = u.shape[-2] > u.shape[-1]
    x = u.transpose(-1, -2) if tall else u
    x = x / x.double().square().sum((-1, -2), keepdim=True).sqrt().clamp(min=1e-7).to(x.dtype)
    for _ in range(5):
        A = x @ x.transpose(-1, -2)
        x = ABC[0] * x + (ABC[1] * A + ABC[2] * A @ A) @ x
    return x.transpose(-1, -2) if tall else x


def norm(x):
    return x.double().square().sum((-1, -2)).sqrt()


def check_update(p, g, m, new_p, new_m, lr, mu):
    p, g, old = p.double().cpu(), g.double().cpu(), m.double().cpu()
    m = mu * old + g
    off = (new_m.double().cpu() - m).abs()
    # one rounding of the sum, half a step, and mu's own: an fp32 in [0.5, 1) is off by 2^-25 at most, times the old momentum
    # (the first form of this line had 2^-24 (|m| + |g|), which leaves mu's rounding out where m and g cancel)
    held = (off <= 2.0 ** -24 * (m.abs() + torch.finfo(torch.float32).tiny) + 2.0 ** -25 * old.abs()).all()
    assert held
    u = g + mu * new_m.double().cpu()
    step = iteration(u)
    rate = lr * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
    used = m.abs().sum((-1, -2)) > 0                     # an expert that never had rows keeps its weights
    most = rate * (4 * norm(iteration(u.float()).double() - step) + 4 * 2.0 ** -22 * norm(step)) + 2.0 ** -23 * norm(p)
    off = norm(new_p.double().cpu() - (p - rate * step))
    assert (off <= most).all(), (off / most).max()
    assert torch.equal(new_p.cpu()[~used], p.float()[~used])


class Net:
    def __init__(self, n, E, sizes, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
        self.x = r(n, sizes[0]).to(dtype).to(DEV)
        self.target = r(n, sizes[2]).to(dtype).to(DEV)
        self.index = torch.randint(-1, E - 1, (n,), generator=g).to(torch.int32).to(DEV)     # the last expert has no rows
        self.E, self.dtype = E, dtype
        # fp32 master weights; the products take them in `dtype`
        self.w = [(r(E, o, i) / i ** 0.5).to(DEV) for i, o in zip(sizes[:-1], sizes[1:])]
        self.b = [(0.1 * r(E, o)).to(DEV) for o in sizes[1:]]
        self.m = [torch.zeros_like(w) for w in self.w]

    def step(self, check=False):
        plan = expert_plan(self.index, self.E)
        w, b = [t.to(self.dtype) for t in self.w], [t.to(self.dtype) for t in self.b]
        h = expert_linear(self.x, w[0], b[0], plan, "relu")
        y = expert_linear(h, w[1], b[1], plan)
        dy = y - self.target
        dh, dw1, db1 = expert_linear_backward(dy, h, w[1], plan)
        dx, dw0, db0 = expert_linear_backward(dh, self.x, w[0], plan, y=h, activation="relu")
        if check:
            check_layer(self.x, w[0], b[0], h, self.index, True)
            check_layer(h, w[1], b[1], y, self.index, False)
            check_gradients(dy, h, w[1], None, self.index, dh, dw1, db1)
            check_gradients(dh, self.x, w[0], h, self.index, dx, dw0, db0)
        before = [(p.clone(), m.clone()) for p, m in zip(self.w, self.m)] if check else None
        grads = [dw0.float(), dw1.float()]
        for p, g, m in zip(self.w, grads, self.m):
            muon_update(p, g, m, lr=0.05, momentum=0.9, clip_value=1e4)
        if check:
            for (p, m), g, new_p, new_m in zip(before, grads, self.w, self.m):
                check_update(p, g, m, new_p, new_m, 0.05, 0.9)
        return y


CASES = [(700, 6, (63, 32, 4), torch.float32), (3001, 5, (27, 96, 33), torch.float32), (513, 4, (136, 256, 128), torch.bfloat16),
         (900, 3, (64, 48, 40), torch.float16)]


@pytest.mark.parametrize("n,E,sizes,dtype", CASES, ids=str)
def test_steps_of_an_expert_network(n, E, sizes, dtype):
    net = Net(n, E, sizes, dtype, n)
    for _ in range(2):
        net.step(check=True)


@pytest.mark.parametrize("n,E,sizes,dtype", CASES, ids=str)
def test_a_captured_step_replays_what_eager_steps_do(n, E, sizes, dtype):
    eager, graphed = Net(n, E, sizes, dtype, n), Net(n, E, sizes, dtype, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = graphed.step()
    for i in range(4):
        for net in (eager, graphed):                     # other rows for other experts, in place
            net.index.copy_(net.index.roll(i + 1))
        graph.replay()
        want = eager.step()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert all(torch.equal(p, q) for p, q in zip(eager.w + eager.m, graphed.w + graphed.m))


def test_autograd_and_the_update():
    """the same step through torch's autograd gives the same bits"""
    net, other = (Net(700, 6, (63, 32, 4), torch.float32, 3) for _ in range(2))
    w, b = [t.requires_grad_() for t in other.w], [t.requires_grad_() for t in other.b]
    plan = expert_plan(other.index, other.E)
    y = expert_linear(expert_linear(other.x, w[0], b[0], plan, "relu"), w[1], b[1], plan)
    (0.5 * (y - other.target).square()).sum().backward()
    for p, m in zip(w, other.m):
        muon_update(p, p.grad, m, lr=0.05, momentum=0.9, clip_value=1e4)
    net.step()
    assert all(torch.equal(p, q) for p, q in zip(net.w, other.w))


def test_inference_mode():
    """a plan made there serves a training step; an update of tensors made there works"""
    net = Net(300, 4, (63, 32, 4), torch.float32, 8)
    with torch.inference_mode():
        plan = expert_plan(net.index, net.E)
        serving = expert_linear(net.x, net.w[0], net.b[0], plan, "relu")
        p, g, m = (torch.ones(40, 40, device=DEV) * v for v in (1.0, 0.5, 0.0))
        muon_update(p, g, m)
        assert bool((p != 1).any())
    w = net.w[0].clone().requires_grad_()
    y = expert_linear(net.x, w, net.b[0], plan, "relu")
    assert torch.equal(y, serving)
    y.sum().backward()
    _, dw, _ = expert_linear_backward(torch.ones_like(y), net.x, net.w[0], plan, y=y.detach(), activation="relu")
    assert torch.equal(w.grad, dw)
    with torch.inference_mode():
        muon_update(net.w[0], dw, net.m[0])
    assert not torch.equal(net.w[0], w.detach())


@pytest.mark.parametrize("how", ["update", "in place"])
def test_weights_written_between_forward_and_backward_are_noticed(how):
    net = Net(300, 4, (63, 32, 4), torch.float32, 9)
    x = net.x.clone().requires_grad_()
    y = expert_linear(x, net.w[0], net.b[0], expert_plan(net.index, net.E))
    if how == "update":
        muon_update(net.w[0], torch.ones_like(net.w[0]), net.m[0])
    else:
        newton_schulz(net.w[0], out=net.w[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()

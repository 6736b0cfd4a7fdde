"""The expert operators (nerf_amd/expert_ops.py) against their definition in 64 bits.

Tolerances.  An output is a sum of k products.  bf16 and fp16 operands are multiplied exactly and added in fp32, so a result
is off by at most k 2^-23 sum |products| from the additions (twice the half step 2^-24 per addition bounds any order) plus half a
step of the output type.  fp32 operands are three bf16 terms: the dropped products are below 3 2^-24 of each product, the
terms' sums add as above (six additions per product, so 6 k 2^-23 bounds it).  `bound` is that, element by element."""
import numpy as np
import pytest
import torch

from nerf_amd import expert_ops
from nerf_amd.expert_ops import expert_linear, expert_linear_backward, expert_plan

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def tolerance(k, magnitude, value, dtype):
    per = 6 * k + 3 if dtype == torch.float32 else k
    tiny = torch.finfo(dtype).tiny       # below it a result's step no longer shrinks with it
    return per * 2.0 ** -23 * magnitude + torch.finfo(dtype).eps / 2 * (value.abs() + tiny)


def index_of(n, E, kind, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "uniform":
        i = rng.integers(0, E, n)
    elif kind == "one":                  # every row with one expert
        i = np.full(n, E - 1)
    elif kind == "none":
        i = np.full(n, -1)
    elif kind == "outside":              # a third of no expert, on either side of the range
        i = rng.integers(-E // 2 - 1, E + E // 2 + 1, n)
    else:                                # "skew": few popular experts, many without rows
        i = (E * rng.random(n) ** 6).astype(np.int64)
    return torch.from_numpy(i.astype(np.int32)).to(DEV)


def plan_by_definition(index, E):
    i = index.cpu().numpy().astype(np.int64)
    key = np.where((i >= 0) & (i < E), i, E)
    counts = np.bincount(key, minlength=E + 1)[:E]
    return counts, np.concatenate([[0], np.cumsum(counts)]), np.argsort(key, kind="stable")


@pytest.mark.parametrize("n,E", [(0, 3), (1, 1), (2, 5), (63, 1), (64, 2), (65, 4096), (1000, 7), (8192, 64), (8193, 64),
                                 (8193, 4096), (40000, 4097), (5000, 16384), (100003, 16384), (300001, 1), (1200007, 4096)])
@pytest.mark.parametrize("kind", ["uniform", "skew", "outside"])
def test_plan(n, E, kind):
    index = index_of(n, E, kind, n + E)
    plan = expert_plan(index, E)
    counts, offsets, order = plan_by_definition(index, E)
    assert np.array_equal(plan.counts.cpu().numpy(), counts)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    # the tile tables: every grouped place, the rows of no expert among them, in exactly one run of one expert; runs of half
    # the length and less last
    at = expert_ops._up4(E) + expert_ops._up4(E + 1) + expert_ops._up4(n)
    runs = plan.buffer[at:at + 8].view(4, 2).tolist()
    at += 8
    ends = np.concatenate([offsets, [n]])
    for shift, (longs, count) in zip((5, 6, 7, 8), runs):
        assert count == (-(-np.diff(ends) // (1 << shift))).sum() <= (n >> shift) + E + 1
        table = plan.buffer[at:at + 2 * count].view(-1, 2).cpu().numpy().astype(np.int64)
        at += expert_ops._up4(2 * ((n >> shift) + E + 1))
        first, rows, expert = table[:, 0], table[:, 1] >> 16, table[:, 1] & 0xffff
        assert (rows > 0).all() and (rows <= 1 << shift).all() and (2 * rows[:longs] > 1 << shift).all() and (2 * rows[longs:] <= 1 << shift).all()
        assert (np.diff(first[:longs]) > 0).all() and (np.diff(first[longs:]) > 0).all()
        grouped = np.argsort(first)
        assert rows.sum() == n and np.array_equal(first[grouped], np.cumsum(rows[grouped]) - rows[grouped])
        assert (first >= ends[expert]).all() and (first + rows <= ends[expert + 1]).all()


@pytest.mark.parametrize("n,E,kind", [(1600009, 4096, "outside"), (2000003, 70, "skew"), (9000011, 300, "skew"), (9000011, 2, "one")])
def test_plan_of_long_chunks(n, E, kind):
    test_plan(n, E, kind)


@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("n", [130, 20000])
def test_plan_of_one_or_no_expert(n, kind):
    index = index_of(n, 9, kind)
    plan = expert_plan(index, 9)
    counts, offsets, order = plan_by_definition(index, 9)
    assert np.array_equal(plan.counts.cpu().numpy(), counts) and np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)


def layer(n, E, k, m, dtype, seed=0, kind="uniform"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g).to(dtype).to(DEV)
    w = (torch.randn(E, m, k, generator=g) / k ** 0.5).to(dtype).to(DEV)
    b = torch.randn(E, m, generator=g).to(dtype).to(DEV)
    dy = torch.randn(n, m, generator=g).to(dtype).to(DEV)
    return x, w, b, dy, index_of(n, E, kind, seed)


def linear64(x, w, b, index, relu):
    """(outputs, sums of the products' magnitudes)"""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    x, w, i = x.double().cpu(), w.double().cpu(), index.cpu()
    b = torch.zeros(w.shape[:2], dtype=torch.float64) if b is None else b.double().cpu()
    for e in range(w.shape[0]):
        r = (i == e).nonzero().flatten()
        y[r] = x[r] @ w[e].T + b[e]
        mag[r] = x[r].abs() @ w[e].abs().T + b[e].abs()
    return (y.clamp(min=0) if relu else y), mag


def backward64(dy, x, w, y, index, relu):
    dz = dy.double().cpu()
    if relu:
        dz = dz * (y.double().cpu() > 0)
    x, w, i = x.double().cpu(), w.double().cpu(), index.cpu()
    out = [torch.zeros_like(x), torch.zeros_like(w), torch.zeros(w.shape[:2], dtype=torch.float64)]
    mag = [torch.zeros_like(o) for o in out]
    rows = 1
    for e in range(w.shape[0]):
        r = (i == e).nonzero().flatten()
        rows = max(rows, r.numel())
        out[0][r], mag[0][r] = dz[r] @ w[e], dz[r].abs() @ w[e].abs()
        out[1][e], mag[1][e] = dz[r].T @ x[r], dz[r].abs().T @ x[r].abs()
        out[2][e], mag[2][e] = dz[r].sum(0), dz[r].abs().sum(0)
    return out, mag, rows


SHAPES = [  # n, E, n_in, n_out, kind
    (1, 1, 1, 1, "uniform"), (1, 4, 64, 32, "uniform"), (7, 3, 5, 3, "uniform"), (48, 32, 256, 128, "skew"),
    (33, 2, 63, 32, "uniform"), (300, 5, 32, 32, "outside"), (1000, 64, 63, 32, "skew"), (2000, 3, 319, 256, "uniform"),
    (129, 2, 130, 257, "one"), (64, 3, 16, 8, "none"), (2500, 8, 96, 100, "skew"), (515, 1, 1024, 40, "uniform"),
    (700, 2, 512, 640, "uniform"), (900, 3, 264, 136, "outside"), (1300, 2, 128, 520, "skew"), (5000, 1, 136, 128, "one"),
    (640, 8, 200, 328, "skew"), (700, 3, 256, 131, "outside"), (3000, 2, 136, 517, "skew"), (300, 4, 131, 259, "uniform"),
    (90, 2, 777, 129, "outside"), (600, 2, 129, 128, "one"), (1500, 70, 136, 128, "skew"), (2000, 90, 100, 70, "outside"),
    (3000, 1000, 63, 32, "skew"), (300, 100, 130, 257, "skew"),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("relu,with_bias", [(False, True), (True, True), (False, False)])
def test_linear(shape, dtype, relu, with_bias):
    n, E, k, m, kind = shape
    x, w, b, _, index = layer(n, E, k, m, DT[dtype], n + m, kind)
    b = b if with_bias else None
    y = expert_linear(x, w, b, expert_plan(index, E), activation="relu" if relu else "none")
    want, mag = linear64(x, w, b, index, relu)
    assert y.dtype == DT[dtype] and tuple(y.shape) == (n, m)
    assert ((y.double().cpu() - want).abs() <= tolerance(k + 1, mag, want, DT[dtype])).all()
    none = (index.cpu() < 0) | (index.cpu() >= E)
    assert (y.cpu()[none] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("relu", [False, True])
def test_backward(shape, dtype, relu):
    n, E, k, m, kind = shape
    x, w, b, dy, index = layer(n, E, k, m, DT[dtype], n + k, kind)
    plan = expert_plan(index, E)
    act = "relu" if relu else "none"
    y = expert_linear(x, w, b, plan, activation=act)
    got = expert_linear_backward(dy, x, w, plan, y=y, activation=act)
    again = expert_linear_backward(dy, x, w, plan, y=y, activation=act)
    want, mag, rows = backward64(dy, x, w, y, index, relu)
    for name, g, a, v, s, count in zip(("x", "weight", "bias"), got, again, want, mag, (m, rows, rows)):
        assert torch.equal(g, a), name                       # the same bits on every run
        assert g.dtype == DT[dtype] and g.shape == v.shape
        assert ((g.double().cpu() - v).abs() <= tolerance(count, s, v, DT[dtype])).all(), name
    only = expert_linear_backward(dy, x, w, plan, y=y, activation=act, want_weight=False, want_bias=False)
    assert torch.equal(only[0], got[0]) and only[1] is None and only[2] is None


def test_gradients_against_differences():
    """f = sum(c * y) in fp32: its change along a direction against the gradients' product with it.  A central difference
    of a function that is linear in each argument alone has no truncation error, so what is left is rounding: y's 2^-24
    relative steps and the products' (tolerance above), summed over the outputs and divided by 2 h."""
    n, E, k, m = 200, 4, 24, 20
    x, w, b, _, index = layer(n, E, k, m, torch.float32, 5, "outside")
    plan = expert_plan(index, E)
    c = torch.randn(n, m, generator=torch.Generator().manual_seed(9)).to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    (expert_linear(*leaves, plan) * c).sum().backward()
    grads, gmag, rows = backward64(c, x, w, None, index, False)
    h = 0.5
    for at in range(3):
        d = torch.randn(leaves[at].shape, generator=torch.Generator().manual_seed(at)).to(DEV)
        ends, slack = [], 0.0
        for sign in (1, -1):
            args = [t.detach() + (sign * h * d if i == at else 0) for i, t in enumerate(leaves)]
            y = expert_linear(*args, plan)
            _, mag = linear64(*args, index, False)
            # the moved argument itself is rounded: 2^-24 of it, inside the products' magnitudes
            slack += float((c.double().cpu().abs() * ((6 * k + 5) * 2.0 ** -23 * mag)).sum())
            ends.append(float((y.double() * c.double()).sum()))
        diff = (ends[0] - ends[1]) / (2 * h)
        dot = float((leaves[at].grad.double() * d.double()).sum())
        off = tolerance((m, rows, rows)[at], gmag[at], grads[at], torch.float32)
        assert abs(diff - dot) <= slack / (2 * h) + float((off * d.double().cpu().abs()).sum())


def test_autograd_matches_the_explicit_backward():
    x, w, b, dy, index = layer(500, 6, 40, 24, torch.bfloat16, 3, "outside")
    plan = expert_plan(index, 6)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = expert_linear(*leaves, plan, activation="relu")
    got = torch.autograd.grad(y, leaves, dy)
    want = expert_linear_backward(dy, x, w, plan, y=y.detach(), activation="relu")
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    y = expert_linear(x, leaves[1], b, plan)                  # weights alone
    assert torch.equal(torch.autograd.grad(y, leaves[1], dy)[0], expert_linear_backward(dy, x, w, plan)[1])
    y = expert_linear(x, w, leaves[2], plan)                  # biases alone
    assert torch.equal(torch.autograd.grad(y, leaves[2], dy)[0], expert_linear_backward(dy, x, w, plan)[2])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_views_and_odd_alignment(dtype):
    """Transposed, strided and odd-offset tensors give the bits of their contiguous copies."""
    n, E, k, m = 90, 3, 37, 29
    x, w, b, dy, index = layer(n, E, k, m, DT[dtype], 1)
    plan = expert_plan(index, E)
    want = expert_linear(x, w, b, plan)
    grads = expert_linear_backward(dy, x, w, plan)
    flat = torch.zeros(x.numel() + w.numel() + 3, dtype=DT[dtype], device=DEV)
    x1 = flat[1:1 + x.numel()].view(n, k)
    x1.copy_(x)
    w1 = flat[2 + x.numel():2 + x.numel() + w.numel()].view(E, m, k)
    w1.copy_(w)
    assert torch.equal(expert_linear(x1, w1, b, plan), want)
    assert all(torch.equal(a, v) for a, v in zip(expert_linear_backward(dy, x1, w1, plan), grads))
    x2, w2, dy2 = x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), dy.t().contiguous().t()
    assert torch.equal(expert_linear(x2, w2, b, plan), want)
    assert all(torch.equal(a, v) for a, v in zip(expert_linear_backward(dy2, x2, w2, plan), grads))
    strided = torch.stack([index, index + 1], 1)[:, 0]
    assert torch.equal(expert_plan(strided, E).order, plan.order)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    n, E, k, m = 100, 3, 70, 40
    x, w, b, dy, index = layer(n, E, k, m, DT[dtype], 2)
    plan = expert_plan(index, E)
    clean = expert_linear(x, w, b, plan, activation="relu")
    x[17, 5], x[40, 0] = float("nan"), float("inf")
    y = expert_linear(x, w, b, plan, activation="relu")
    others = [i for i in range(n) if i not in (17, 40)]
    assert torch.equal(y[others], clean[others]) and torch.isnan(y[17]).all()
    # a gradient that is not finite behind the relu, and in a row of no expert, reaches nothing
    x, w, b, dy, index = layer(n, E, k, m, DT[dtype], 2)
    index[3] = -1
    plan = expert_plan(index, E)
    y = expert_linear(x, w, b, plan, activation="relu")
    want = expert_linear_backward(torch.where(y > 0, dy, 0), x, w, plan)
    dy = torch.where(y > 0, dy, float("nan"))
    x[3] = float("nan")
    got = expert_linear_backward(dy, x, w, plan, y=y, activation="relu")
    assert all(torch.equal(a, v) for a, v in zip(got, want))


def test_a_run_of_layers_on_a_side_stream_and_in_a_graph():
    """Plan, two layers, their gradients: eager, on another stream, and captured and replayed with new contents."""
    n, E, k, h, m = 400, 6, 63, 48, 4
    x, w1, b1, _, index = layer(n, E, k, h, torch.float32, 4, "skew")
    _, w2, b2, dy, _ = layer(n, E, h, m, torch.float32, 6)

    def step(x, index, dy):
        with torch.no_grad():
            plan = expert_plan(index, E)
            z = expert_linear(x, w1, b1, plan, activation="relu")
            y = expert_linear(z, w2, b2, plan)
            dz, dw2, db2 = expert_linear_backward(dy, z, w2, plan)
            dx, dw1, db1 = expert_linear_backward(dz, x, w1, plan, y=z, activation="relu")
            return y, dx, dw1, db1, dw2, db2

    want = step(x, index, dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, index, dy)
    side.synchronize()
    assert all(torch.equal(a, v) for a, v in zip(got, want))
    xs, index_s, dys = x.clone(), index.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, index_s, dys)
    for seed in range(3):
        x2, _, _, _, index2 = layer(n, E, k, h, torch.float32, 20 + seed, "outside" if seed else "skew")
        dy2 = torch.randn(n, m, generator=torch.Generator().manual_seed(seed)).to(DEV)
        xs.copy_(x2), index_s.copy_(index2), dys.copy_(dy2)
        graph.replay()
        torch.cuda.synchronize()
        want = step(x2, index2, dy2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, v) for a, v in zip(out, want))


def test_autograd_under_capture_is_refused():
    x, w, b, _, index = layer(40, 2, 8, 8, torch.float32, 0)
    plan = expert_plan(index, 2)
    w.requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(expert_ops.NrfError, match="capture"):
            expert_linear(x, w, b, plan)
        keep = torch.zeros(1, device=DEV)   # the captured graph holds one node
    graph.replay()
    torch.cuda.synchronize()
    assert float(keep) == 0


@pytest.mark.parametrize("n,n_in,n_out,dtype", [(4194300, 512, 128, "bf16"), (4200003, 520, 136, "fp16"), (34000001, 64, 5, "fp32")])
def test_offsets_past_32_bits(n, n_in, n_out, dtype):
    """x of 2^31 elements and more (the wide kernels up to there, the general tile beyond); rows sampled, dW over all of them in 64 bits"""
    g = torch.Generator(device=DEV).manual_seed(n)
    x = torch.randn(n, n_in, device=DEV, generator=g, dtype=DT[dtype])
    w = torch.randn(3, n_out, n_in, device=DEV, generator=g).to(DT[dtype])
    index = torch.randint(-1, 3, (n,), device=DEV, generator=g, dtype=torch.int32)
    plan = expert_plan(index, 3)
    y = expert_linear(x, w, None, plan)
    dy = torch.randn(n, n_out, device=DEV, generator=g, dtype=DT[dtype])
    dx, dw, _ = expert_linear_backward(dy, x, w, plan)
    at = torch.cat([torch.arange(64), torch.randint(0, n, (500,)), torch.arange(n - 64, n)]).to(DEV)
    want, mag = linear64(x[at], w, None, index[at], False)
    assert ((y[at].double().cpu() - want).abs() <= tolerance(n_in, mag, want, DT[dtype])).all()
    (want, _, _), (mag, _, _), _ = backward64(dy[at], x[at], w, None, index[at], False)
    assert ((dx[at].double().cpu() - want).abs() <= tolerance(n_out, mag, want, DT[dtype])).all()
    for e in range(3):
        want, mag = (torch.zeros(n_out, n_in, dtype=torch.float64, device=DEV) for _ in range(2))
        for r in range(0, n, 1 << 20):
            part = dy[r:r + (1 << 20)].double() * (index[r:r + (1 << 20)] == e)[:, None]
            rows = x[r:r + (1 << 20)].double()
            want += part.T.contiguous() @ rows
            mag += part.T.abs().contiguous() @ rows.abs()
        off = (dw[e].double() - want).abs()
        assert (off <= tolerance(n, mag, want, DT[dtype])).all()
        assert float(off.norm() / want.norm()) <= 2.0 ** -8     # far under what the bound over so many rows allows


@pytest.mark.parametrize("n_in,n_out,dtype", [(63, 32, "fp32"), (130, 70, "fp32"), (256, 128, "bf16"), (100, 9, "fp16")])
@pytest.mark.parametrize("relu", [False, True])
def test_a_batch_without_rows(n_in, n_out, dtype, relu):
    x, w = torch.zeros(0, n_in, dtype=DT[dtype], device=DEV), torch.randn(5, n_out, n_in, device=DEV).to(DT[dtype])
    plan, act = expert_plan(torch.zeros(0, dtype=torch.int32, device=DEV), 5), "relu" if relu else "none"
    y = expert_linear(x, w, w[:, :, 0], plan, act)
    dx, dw, db = expert_linear_backward(y, x, w, plan, y=y, activation=act)
    assert y.shape == (0, n_out) and dx.shape == x.shape and plan.counts.sum() == 0 and not plan.offsets.any()
    assert dw.shape == w.shape and not dw.any() and db.shape == (5, n_out) and not db.any()


def test_index_values_of_any_size():
    index = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, 3, 2, -1, 65536, 131074, 2, 16384 * 2 + 1], dtype=torch.int32, device=DEV)
    plan = expert_plan(index, 3)
    assert plan.counts.tolist() == [1, 0, 2] and plan.offsets.tolist() == [0, 1, 1, 3]
    assert plan.order.tolist() == [2, 4, 8, 0, 1, 3, 5, 6, 7, 9]


def test_a_plan_written_to_between_forward_and_backward_is_noticed():
    x = torch.randn(20, 8, device=DEV, requires_grad=True)
    plan = expert_plan(torch.zeros(20, dtype=torch.int32, device=DEV), 2)
    y = expert_linear(x, torch.randn(2, 4, 8, device=DEV), None, plan)
    plan.order.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals():
    x, w, b, dy, index = layer(40, 2, 8, 6, torch.float32, 0)
    plan = expert_plan(index, 2)
    E = expert_ops.NrfError
    for bad in (index.long(), index.view(2, 20), index.cpu()):
        with pytest.raises(E):
            expert_plan(bad, 2)
    for experts in (0, -1, 16385):
        with pytest.raises(E):
            expert_plan(index, experts)
    for args in ((x[:39], w, b, plan), (x, w[:1], b, plan), (x, w, b[:, :5], plan), (x, w[:, :, :7], b, plan),
                 (x.double(), w.double(), b.double(), plan), (x, w.bfloat16(), b, plan), (x, w, b.cpu(), plan), (x, w, b, index)):
        with pytest.raises(E):
            expert_linear(*args)
    with pytest.raises(E):
        expert_linear(x, w, b, plan, activation="gelu")
    with pytest.raises(E):
        expert_linear_backward(dy, x, w, plan, activation="relu")
    with pytest.raises(E):
        expert_linear_backward(dy[:, :5], x, w, plan)
    with pytest.raises(E):
        expert_linear_backward(dy, x, w, plan, want_weight=False)

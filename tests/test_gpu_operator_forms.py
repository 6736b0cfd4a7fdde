"""The kernel forms of the expert products and of the update that only larger shapes reach, with odd remainders in every
dimension.  Each shape names the forms that it is there for, and they are looked up among the kernels that ran: a rule that
sends a shape elsewhere is noticed.

Tolerances as in test_gpu_experts.py (k products: 2^-23 k of their magnitudes, six times that for three bf16 terms, and half a
step of the output) and test_gpu_muon.py (four times what the iteration in fp32 is off)."""
import re

import pytest
import torch
from test_gpu_experts import DEV, DT, backward64, layer, linear64, tolerance
from test_gpu_muon import bound, definition, gradient, muon64, norm

from nerf_amd.expert_ops import expert_linear, expert_linear_backward, expert_plan
from nerf_amd.muon_ops import muon_update, newton_schulz

pytestmark = pytest.mark.gpu


def form(name):
    """'expert_tile Fp32 1 128' of a kernel's name, demangled or not; None for others"""
    found = re.search(r"((?:expert|schulz)_\w+?)_kernel", name)
    if not found:
        return None
    rest = name[found.end():]
    if rest.startswith("<"):
        args = rest[1:rest.index(">(")].replace("(anonymous namespace)::", "").split(", ")
    else:
        args = [a or b for a, b in re.findall(r"NS_\d+(\w+?)E|L[ib](\d+)E", rest)]
    return " ".join([found.group(1)] + args)


def forms(call):
    from torch.profiler import ProfilerActivity, profile
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    return {form(e.name).replace("false", "0").replace("true", "1") for e in prof.events() if form(e.name)}


def check_forms(call, wanted):
    """each of `wanted` begins the name of a form that ran"""
    ran = forms(call)
    if not ran:
        pytest.skip("the profiler recorded no kernel here: which forms ran is not known")
    assert all(any(r.startswith(f) for r in ran) for f in wanted), ran


def test_names_of_kernels():
    assert form("void (anonymous namespace)::expert_tile_kernel<(anonymous namespace)::Fp32, 1, 128>((anonymous namespace)::ExpertArgs, int, int)") == "expert_tile Fp32 1 128"
    assert form("_ZN12_GLOBAL__N_121schulz_product_kernelINS_5Out32ELi2ELi128EEEvNS_10SchulzArgsENS_10LargeShapeEPDF16_iiii").startswith("schulz_product Out32 2 128")
    assert form("void at::native::vectorized_elementwise_kernel<4, foo>(int)") is None


# n, E, n_in, n_out, kind, dtype, forms (forward 0, dx 1, dW 2)
EXPERTS = [
    (20011, 8, 319, 300, "uniform", "fp32", ["expert_tile Fp32 0 128"]),
    (20011, 8, 319, 256, "uniform", "fp32", ["expert_tile Fp32 1 128", "expert_tile Fp32 2 128", "expert_sum Fp32 0"]),
    (20011, 8, 319, 253, "outside", "fp16", ["expert_tile Fp16 1 128", "expert_tile Fp16 2 128", "expert_sum Fp16"]),
    (3001, 16, 1001, 1003, "skew", "fp32", ["expert_tile Fp32 2 128"]),
    (3001, 16, 1001, 1003, "skew", "bf16", ["expert_tile Bf16 2 128"]),
    (16411, 8, 515, 513, "uniform", "fp16", ["expert_tile Fp16 0 64", "expert_tile Fp16 1 64", "expert_tile Fp16 2 128"]),
    (4003, 8, 1001, 1001, "uniform", "fp16", ["expert_tile Fp16 2 64"]),
    (43007, 8, 200, 520, "skew", "bf16", ["expert_wide_rows Bf16 0 256", "expert_wide_rows Bf16 1 128", "expert_wide_dw Bf16", "expert_mask Bf16", "expert_sum Bf16"]),
    (43007, 8, 200, 520, "outside", "fp16", ["expert_wide_rows Fp16 0 256", "expert_wide_rows Fp16 1 128", "expert_wide_dw Fp16", "expert_mask Fp16"]),
    (44003, 6, 328, 517, "uniform", "fp16", ["expert_wide_rows Fp16 0 256", "expert_tile Fp16 2 128"]),
    (900, 12, 776, 648, "uniform", "bf16", ["expert_wide_rows Bf16 0 128", "expert_wide_dw Bf16"]),
    (5003, 3, 63, 31, "skew", "bf16", ["expert_tile Bf16 0 64", "expert_tile Bf16 1 64", "expert_tile Bf16 2 64"]),
    (2003, 40, 63, 31, "skew", "fp32", ["expert_cell_forward 2 1", "expert_cell_backward 2 1"]),
    (2003, 40, 64, 33, "skew", "fp32", ["expert_cell_forward 2 2", "expert_cell_backward 2 2"]),
    (2003, 40, 31, 33, "skew", "fp32", ["expert_cell_forward 1 2", "expert_cell_backward 1 2"]),
    (70001, 2, 33, 41, "uniform", "fp32", ["expert_cell_backward 2 2", "expert_sum Fp32 1"]),
    (2003, 40, 31, 32, "skew", "fp32", ["expert_cell_forward 1 1", "expert_cell_backward 1 1"]),
]


@pytest.mark.parametrize("n,E,k,m,kind,dtype,wanted", EXPERTS, ids=lambda v: str(v) if not isinstance(v, list) else "")
def test_experts(n, E, k, m, kind, dtype, wanted):
    x, w, b, dy, index = layer(n, E, k, m, DT[dtype], n + m, kind)
    plan = expert_plan(index, E)
    y = expert_linear(x, w, b, plan, activation="relu")
    want, mag = linear64(x, w, b, index, True)
    assert ((y.double().cpu() - want).abs() <= tolerance(k + 1, mag, want, DT[dtype])).all()
    assert not y.cpu()[(index.cpu() < 0) | (index.cpu() >= E)].any()
    got = expert_linear_backward(dy, x, w, plan, y=y, activation="relu")
    again = expert_linear_backward(dy, x, w, plan, y=y, activation="relu")
    want, mag, rows = backward64(dy, x, w, y, index, True)
    for name, g, a, v, s, count in zip(("x", "weight", "bias"), got, again, want, mag, (m, rows, rows)):
        assert torch.equal(g, a), name
        assert ((g.double().cpu() - v).abs() <= tolerance(count, s, v, DT[dtype])).all(), name
    check_forms(lambda: (expert_linear(x, w, b, plan, activation="relu"), expert_linear_backward(dy, x, w, plan, y=y, activation="relu")), wanted)


# products: A 0, Q 1, X' 2, the last X' 3, A in parts 4
UPDATES = [
    ((2, 1000, 4000), "fp32", ["schulz_product Out32 2 128", "schulz_product Out32 3 128", "schulz_product Out32 4 128"]),
    ((2, 4001, 997), "bf16", ["schulz_product Out32 2 128", "schulz_product OutBf16 3 128"]),
    ((6, 1001, 1030), "fp16", ["schulz_product Out32 0 128", "schulz_product Out32 1 128", "schulz_product OutFp16 3 128"]),
    ((3, 520, 700), "fp32", ["schulz_product Out32 2 64", "schulz_product Out32 3 64"]),
    ((2, 128, 283), "fp32", ["schulz_step Out32 8 0", "schulz_step Out32 8 1"]),
    ((1, 63, 600), "bf16", ["schulz_step Out32 4 0", "schulz_step OutBf16 4 1"]),
    ((5, 100, 150), "fp32", ["schulz_block Out32 8"]),
    ((5, 60, 510), "fp16", ["schulz_block OutFp16 4"]),
    ((9, 30, 120), "fp32", ["schulz_small Out32 4 0"]),
    ((9, 120, 30), "fp32", ["schulz_small Out32 4 1"]),
]


@pytest.mark.parametrize("shape,dtype,wanted", UPDATES, ids=lambda v: str(v) if not isinstance(v, list) else "")
def test_newton_schulz(shape, dtype, wanted):
    g = gradient(*shape, seed=sum(shape), dtype=DT[dtype], scale=1.0 if dtype == "fp16" else 1e-3)
    on = g.to(DEV)
    got = newton_schulz(on)
    want = definition(g)
    off, most = norm(got.double().cpu() - want), bound(g, want, DT[dtype])
    assert (off <= most).all(), (off / most).max()
    assert torch.equal(got, newton_schulz(on))
    check_forms(lambda: newton_schulz(on), wanted)


@pytest.mark.parametrize("shape,wanted", [((2, 1001, 3999), "schulz_product OutMuon 3 128"), ((2, 3999, 1001), "schulz_product OutMuon 3 128"),
                                          ((2, 128, 283), "schulz_step OutMuon 8 1"), ((2, 600, 63), "schulz_step OutMuon 4 1"),
                                          ((3, 317, 99), "schulz_step OutMuon 8 1"), ((3, 90, 111), "schulz_block OutMuon 8")], ids=str)
def test_muon_update(shape, wanted):
    gen = torch.Generator().manual_seed(7)
    p, m = torch.randn(shape, generator=gen) / shape[2] ** 0.5, 2e-3 * torch.randn(shape, generator=gen)
    g = gradient(*shape, seed=10)
    pd, md, gd = p.to(DEV), m.to(DEV), g.to(DEV)
    options = dict(lr=0.1, weight_decay=0.3, clip_value=2e-3, grad_scale=0.5, momentum=0.9)
    muon_update(pd, gd, md, **options)
    p64, m64, o = muon64(p, g, m, 0.1, 0.9, True, 0.3, 2e-3, 0.5)
    _, _, o32 = muon64(p, g, m, 0.1, 0.9, True, 0.3, 2e-3, 0.5, torch.float32)
    # as in test_gpu_muon.py: half a step of the result, of mu times the old momentum and of g
    assert ((md.double().cpu() - m64).abs() <= 2.0 ** -24 * (m64.abs() + 2 * m.double().abs() + 2e-3)).all()
    rate = 0.1 * max(1.0, shape[1] / shape[2]) ** 0.5
    off = rate * (4 * norm(o32.double() - o) + 4 * 2.0 ** -22 * norm(o)) + 5 * 2.0 ** -24 * (norm(p64) + rate * norm(o))
    assert (norm(pd.double().cpu() - p64) <= off).all()
    check_forms(lambda: muon_update(pd, gd, md, **options), [wanted])

"""What torch cannot follow through the library is refused: forward-mode derivatives and torch.jit.trace.  The library's call
is replaced by the same layer in torch, with its outputs written as the kernels write them (behind torch's back), so that the
wrappers run without a GPU; a call that is not refused would return a tangent of None, or a trace of the empty output."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from nerf_amd import expert_ops, muon_ops
from nerf_amd._lib import NrfError

N, E, K, M = 6, 2, 3, 4
INDEX = torch.tensor([0, 1, 1, -1, 0, 1], dtype=torch.int32)


class _Plan(expert_ops.ExpertPlan):
    def __init__(self):
        super().__init__(torch.zeros(8, dtype=torch.int32), N, E)


def _layer(x, weight, bias, plan, activation):
    y = torch.empty((x.shape[0], weight.shape[1]), dtype=x.dtype)
    x, weight = x.detach().contiguous().numpy(), weight.detach().contiguous().numpy()
    for i, e in enumerate(INDEX.tolist()):
        y.numpy()[i] = weight[e] @ x[i] + (0 if bias is None else bias.detach().numpy()[e]) if e >= 0 else 0
    if activation == "relu":
        np.maximum(y.numpy(), 0, out=y.numpy())
    return y


@pytest.fixture
def layer(monkeypatch):
    monkeypatch.setattr(expert_ops, "_check_layer", lambda *a: None)
    monkeypatch.setattr(expert_ops, "_forward", _layer)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    g = torch.Generator().manual_seed(0)
    return torch.randn(N, K, generator=g), torch.randn(E, M, K, generator=g), torch.randn(E, M, generator=g), _Plan()


@pytest.mark.parametrize("at", [0, 1, 2])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(layer, at, requires_grad):
    args = [t.requires_grad_(requires_grad) for t in layer[:3]]
    with forward_ad.dual_level():
        want = _layer(*args, layer[3], "relu")
        assert torch.equal(expert_ops.expert_linear(*args, layer[3], "relu"), want)      # a level without tangents changes nothing
        args[at] = forward_ad.make_dual(args[at].detach(), torch.ones_like(args[at]))
        for context in (torch.enable_grad, torch.no_grad):
            with context(), pytest.raises(NrfError, match="forward-mode"):
                expert_ops.expert_linear(*args, layer[3], "relu")
    x, w, b = (t.detach() for t in layer[:3])
    with pytest.raises((NrfError, RuntimeError)):
        torch.func.jvp(lambda t: expert_ops.expert_linear(t, w, b, layer[3]), (x,), (torch.ones_like(x),))


def test_a_trace_is_refused(layer):
    x, w, b, plan = layer
    with pytest.raises(NrfError, match="trace"):
        torch.jit.trace(lambda t: expert_ops.expert_linear(t, w, b, plan), (x,), check_trace=False)


def test_the_other_operators_refuse_both():
    x, plan = torch.ones(N, K), _Plan()
    calls = {
        "expert_linear_backward": lambda t: expert_ops.expert_linear_backward(torch.ones(N, M), t, torch.ones(E, M, K), plan)[0],
        "newton_schulz": muon_ops.newton_schulz,
        "muon_update": lambda t: muon_ops.muon_update(torch.ones(N, K), t, torch.ones(N, K)),
    }
    for name, call in calls.items():
        with forward_ad.dual_level():
            with pytest.raises(NrfError, match=f"{name}: forward-mode"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(NrfError, match=f"{name}: torch.jit.trace"):
            torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(NrfError, match="expert_plan: torch.jit.trace"):
        torch.jit.trace(lambda t: expert_ops.expert_plan(t, E).order, (INDEX,), check_trace=False)

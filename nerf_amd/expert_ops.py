"""Tensor-level wrappers over the expert entry points of the C ABI (include/nerf_amd.h, nrf_expert_*): rows grouped by
expert, the product of every row with its expert's weights, and the gradients.  torch only owns the memory; all arithmetic
happens in libnerf_amd.so.

The KiloNeRF kernels (``kilo_ops``) are the fused form for one fixed tiny network per cell; these take any layer size, fp32,
bf16 or fp16, and up to 16384 experts."""
from __future__ import annotations

import contextlib
import ctypes as C

import torch
from torch.autograd import forward_ad

from ._lib import NrfError, check, lib
from .ops import _ptr

MAX_EXPERTS = 16384
MAX_ROWS = 1 << 28
MAX_WIDTH = 65536
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # the C ABI's NRF_DTYPE_*
ACTIVATIONS = {"none": 0, "relu": 1}                               # NRF_ACT_*


# What a call costs the host counts here: grouping 2048 rows takes the GPU 6 us.
_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """the context of work on ``device``; nothing to switch (1.3 us) where it is current"""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(t: torch.Tensor):
    """the current stream of the tensor's device, without building a Stream object (2 us)"""
    return C.c_void_p(torch._C._cuda_getCurrentRawStream(t.device.index))


def _refuse_unseen(name: str, *tensors) -> None:
    """What torch cannot see pass through the library: a trace would record the empty output alone, a tangent of forward-mode
    differentiation would be dropped, which torch takes for zero."""
    if torch._C._is_tracing():
        raise NrfError(f"{name}: torch.jit.trace does not see the library's kernels (the traced graph would return memory that "
                       "nothing wrote)")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NrfError(f"{name}: forward-mode derivatives (dual tensors) are not supported")


def _up4(v: int) -> int:
    return (v + 3) & ~3


class ExpertPlan:
    """Which rows belong to which expert (``expert_plan``).  ``counts`` (E,), ``offsets`` (E + 1,) and ``order`` (n,) are
    int32 views of the plan's buffer: expert e's rows are ``order[offsets[e]:offsets[e + 1]]``, ascending; the rows of no
    expert stand behind ``offsets[E]``."""

    def __init__(self, buffer: torch.Tensor, n_rows: int, num_experts: int):
        self.buffer, self.n_rows, self.num_experts = buffer, n_rows, num_experts
        self.device = buffer.device

    @property
    def counts(self) -> torch.Tensor:
        return self.buffer[:self.num_experts]

    @property
    def offsets(self) -> torch.Tensor:
        at = _up4(self.num_experts)
        return self.buffer[at:at + self.num_experts + 1]

    @property
    def order(self) -> torch.Tensor:
        at = _up4(self.num_experts) + _up4(self.num_experts + 1)
        return self.buffer[at:at + self.n_rows]


def expert_plan(index: torch.Tensor, num_experts: int) -> ExpertPlan:
    """Group the rows of a batch by expert (nrf_expert_plan).  ``index`` (n,) int32 on the GPU: the expert of each row; a
    value outside [0, num_experts) means the row has none.  Nothing is read back, the result is the same on every run."""
    _refuse_unseen("expert_plan")
    if not index.is_cuda:
        raise NrfError("index: expected a cuda tensor (there is no CPU fallback)")
    if index.dtype != torch.int32 or index.ndim != 1:
        raise NrfError(f"index: expected a one-dimensional int32 tensor, got {index.dtype} {tuple(index.shape)}")
    num_experts = int(num_experts)
    n = index.shape[0]
    if not 1 <= num_experts <= MAX_EXPERTS or n > MAX_ROWS:
        raise NrfError(f"expert_plan: {n} rows over {num_experts} experts; 1 to {MAX_EXPERTS} experts and up to {MAX_ROWS} rows are supported")
    index = index.contiguous()
    L = lib()
    plan_bytes, work_bytes = L.nrf_expert_plan_bytes(n, num_experts), L.nrf_expert_plan_workspace_bytes(n, num_experts)
    plan = torch.empty(plan_bytes // 4, dtype=torch.int32, device=index.device)
    work = torch.empty(work_bytes, dtype=torch.uint8, device=index.device) if work_bytes else None
    with _on(index.device):
        check(L.nrf_expert_plan(_ptr(index), n, num_experts, _ptr(plan), plan_bytes, _ptr(work), work_bytes, _stream(index)),
              "nrf_expert_plan")
    return ExpertPlan(plan, n, num_experts)


def _check_layer(x, weight, bias, plan, activation):
    if not isinstance(plan, ExpertPlan):
        raise NrfError("plan: expected an ExpertPlan (expert_plan)")
    if activation not in ACTIVATIONS:
        raise NrfError(f"activation {activation!r}: expected one of {sorted(ACTIVATIONS)}")
    if x.dtype not in DTYPES:
        raise NrfError(f"x: expected float32, bfloat16 or float16, got {x.dtype}")
    if x.ndim != 2 or x.shape[0] != plan.n_rows:
        raise NrfError(f"x: shape {tuple(x.shape)}, want ({plan.n_rows}, n_in) as the plan's rows")
    if weight.ndim != 3 or weight.shape[0] != plan.num_experts or weight.shape[2] != x.shape[1]:
        raise NrfError(f"weight: shape {tuple(weight.shape)}, want ({plan.num_experts}, n_out, {x.shape[1]})")
    if not (1 <= weight.shape[1] <= MAX_WIDTH and 1 <= weight.shape[2] <= MAX_WIDTH):
        raise NrfError(f"weight: {tuple(weight.shape)}; layer sizes of 1 to {MAX_WIDTH} are supported")
    tensors = [("x", x), ("weight", weight)]
    if bias is not None:
        if tuple(bias.shape) != (plan.num_experts, weight.shape[1]):
            raise NrfError(f"bias: shape {tuple(bias.shape)}, want {(plan.num_experts, weight.shape[1])}")
        tensors.append(("bias", bias))
    for name, t in tensors:
        if not t.is_cuda or t.device != plan.device:
            raise NrfError(f"{name}: on {t.device}, the plan on {plan.device} (there is no CPU fallback)")
        if t.dtype != x.dtype:
            raise NrfError(f"{name}: {t.dtype}, x is {x.dtype}")


def _forward(x, weight, bias, plan, activation):
    x, weight = x.contiguous(), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty((x.shape[0], weight.shape[1]), dtype=x.dtype, device=x.device)
    with _on(x.device):
        check(lib().nrf_expert_linear(_ptr(x), _ptr(weight), _ptr(bias), _ptr(plan.buffer), plan.n_rows, plan.num_experts,
                                      x.shape[1], weight.shape[1], DTYPES[x.dtype], ACTIVATIONS[activation], _ptr(y),
                                      _stream(x)), "nrf_expert_linear")
    return y


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, plan, activation):
        y = _forward(x.detach(), weight.detach(), None if bias is None else bias.detach(), plan, activation)
        ctx.plan, ctx.activation = plan, activation
        # the plan's buffer among them: autograd then notices a write to the views that the plan hands out (a buffer made in
        # inference mode counts no writes and cannot be saved)
        ctx.save_for_backward(x, weight, y if activation == "relu" else None, None if plan.buffer.is_inference() else plan.buffer)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        if torch.cuda.is_current_stream_capturing():
            raise NrfError(_CAPTURE)
        x, weight, y, _ = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx, dw, db = expert_linear_backward(grad_y, x, weight, ctx.plan, y=y, activation=ctx.activation, want_x=want_x,
                                            want_weight=want_w or want_b, want_bias=want_b)
        return dx, dw if want_w else None, db, None, None


_CAPTURE = ("expert_linear: autograd under graph capture is refused (a captured backward that meets a live eager graph of "
            "the same leaves ends the process): capture expert_linear under torch.no_grad() and expert_linear_backward")


def expert_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, plan: ExpertPlan,
                  activation: str = "none") -> torch.Tensor:
    """``y[i] = act(weight[index[i]] @ x[i] + bias[index[i]])`` for the rows of ``plan``, zeros for rows of no expert
    (nrf_expert_linear).  x (n, n_in), weight (E, n_out, n_in), bias (E, n_out) or None, all float32, bfloat16 or float16
    alike; ``activation`` "none" or "relu".  Differentiable in x, weight and bias: once, in reverse mode; forward mode and
    ``torch.jit.trace`` are refused."""
    _refuse_unseen("expert_linear", x, weight, bias)
    _check_layer(x, weight, bias, plan, activation)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        if torch.cuda.is_current_stream_capturing():
            raise NrfError(_CAPTURE)
        return _ExpertLinear.apply(x, weight, bias, plan, activation)
    return _forward(x, weight, bias, plan, activation)


@torch.no_grad()
def expert_linear_backward(grad_y: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan,
                           y: torch.Tensor | None = None, activation: str = "none", want_x: bool = True,
                           want_weight: bool = True, want_bias: bool = True):
    """Gradients of ``expert_linear`` -> (grad_x, grad_weight, grad_bias), None for those not wanted
    (nrf_expert_linear_backward).  ``y``: the forward's outputs, needed with "relu".  grad_bias is summed with grad_weight,
    so it needs ``want_weight``.  The same bits on every run.  Not differentiable itself."""
    _refuse_unseen("expert_linear_backward", grad_y, x, weight)
    _check_layer(x, weight, None, plan, activation)
    shape = (x.shape[0], weight.shape[1])
    if activation == "relu" and y is None:
        raise NrfError("expert_linear_backward: relu needs y, the forward's outputs")
    if want_bias and not want_weight:
        raise NrfError("expert_linear_backward: want_bias needs want_weight")
    y = y if activation == "relu" else None
    for name, t in (("grad_y", grad_y), ("y", y)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != x.dtype or t.device != plan.device):
            raise NrfError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, want {x.dtype} {shape} on {plan.device}")
    grad_y, x, weight = grad_y.contiguous(), x.contiguous(), weight.contiguous()
    y = None if y is None else y.contiguous()
    dx = torch.empty_like(x) if want_x else None
    dw = torch.empty_like(weight) if want_weight else None
    db = torch.empty(weight.shape[:2], dtype=x.dtype, device=x.device) if want_bias else None
    L = lib()
    n_in, n_out, dtype = x.shape[1], weight.shape[1], DTYPES[x.dtype]
    need = L.nrf_expert_linear_backward_workspace_bytes(plan.n_rows, plan.num_experts, n_in, n_out, dtype)
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with _on(x.device):
        check(L.nrf_expert_linear_backward(_ptr(grad_y), _ptr(x), _ptr(weight), _ptr(y), _ptr(plan.buffer), plan.n_rows,
                                           plan.num_experts, n_in, n_out, dtype, ACTIVATIONS[activation], _ptr(dx), _ptr(dw),
                                           _ptr(db), _ptr(work), need, _stream(x)), "nrf_expert_linear_backward")
    return dx, dw, db

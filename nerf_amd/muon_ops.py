"""Tensor-level wrappers over the orthogonalised update of the C ABI (include/nerf_amd.h, nrf_newton_schulz and
nrf_muon_update): Newton-Schulz products and the Muon step that stands beside ``ops.clip_adam``.  torch only owns the memory;
all arithmetic happens in libnerf_amd.so."""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import NrfError, check, lib
from .expert_ops import DTYPES, _on, _refuse_unseen, _stream
from .ops import _ptr

COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # steep at 0 (weak directions catch up in five steps), within 0.7 .. 1.2 near 1
MAX_TENSORS = 32                           # of one nrf_muon_update call


def _written(tensors) -> None:
    """the kernels write behind torch's back: autograd's version counters (tensors of inference mode have none)"""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _shared(written, read, size: int) -> bool:
    """whether one of the tensors at ``written``, all of ``size`` bytes, shares memory with another or with one at ``read``"""
    ends = {True: 0, False: 0}     # of what was passed in the order of the addresses: the written, the read
    for at, in_place in sorted([(p, True) for p in written] + [(p, False) for p in read]):
        if at < ends[True] or (in_place and at < ends[False]):
            return True
        ends[in_place] = at + size
    return False


def _workspace(batch: int, rows: int, cols: int, device):
    need = lib().nrf_newton_schulz_workspace_bytes(batch, rows, cols)
    if need < 0:
        raise NrfError(f"{batch} matrices of {rows} x {cols}: sides of 1 to 65536 and up to 65535 matrices are supported "
                       "(2^24 up to 32 x 128, 64 x 544 and 128 x 160), 2^24 tiles of 64 x 64 in all")
    return (torch.empty(need, dtype=torch.uint8, device=device) if need else None), need


@torch.no_grad()
def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Orthogonalise matrices (nrf_newton_schulz): ``X = g / max(|g|_F, eps)``, then ``steps`` times
    ``X <- a X + (b A + c A^2) X`` with ``A = X X^T``.  g (rows, cols) or (batch, rows, cols), float32, bfloat16 or float16;
    fp32-class arithmetic for every type, one rounding at the end.  ``out`` may be ``g``, but share no other memory with it.  Not
    differentiable."""
    _refuse_unseen("newton_schulz", g)
    if not g.is_cuda:
        raise NrfError("g: expected a cuda tensor (there is no CPU fallback)")
    if g.dtype not in DTYPES or g.ndim not in (2, 3):
        raise NrfError(f"g: expected a float32, bfloat16 or float16 matrix or batch of matrices, got {g.dtype} {tuple(g.shape)}")
    rows, cols = g.shape[-2:]
    batch = g.shape[0] if g.ndim == 3 else 1
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    elif out.shape != g.shape or out.dtype != g.dtype or out.device != g.device or not out.is_contiguous():
        raise NrfError(f"out: expected a contiguous {g.dtype} {tuple(g.shape)} on {g.device}")
    work, need = _workspace(batch, rows, cols, g.device)
    g = g.contiguous()
    if 0 < abs(out.data_ptr() - g.data_ptr()) < g.numel() * g.element_size():
        raise NrfError("out: overlaps g without being g (matrices would be read after others were written over them)")
    a, b, c = coefficients
    with _on(g.device):
        check(lib().nrf_newton_schulz(_ptr(g), _ptr(out), batch, rows, cols, DTYPES[g.dtype], int(steps), a, b, c, eps,
                                      _ptr(work), need, _stream(g)), "nrf_newton_schulz")
    _written([out])
    return out


@torch.no_grad()
def muon_update(params, grads, momentum_buffers, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                weight_decay: float = 0.0, clip_value: float = 40.0, grad_scale: float = 1.0, steps: int = 5,
                coefficients=COEFFICIENTS, eps: float = 1e-7) -> None:
    """One Muon step in place (nrf_muon_update) on a float32 tensor (rows, cols) or (batch, rows, cols), or on a list of such
    tensors of one shape (more than 32, or than one call's matrices, go in several calls).  ``momentum_buffers`` like ``params``, zero at the first step:
    ``g = clamp(grad * grad_scale, +-clip_value)``, ``m <- momentum m + g``, ``u = g + momentum m`` (nesterov) or ``m``,
    ``p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) newton_schulz(u)``.  A parameter or momentum buffer shares no
    memory with another tensor of the call; gradients may with each other."""
    if isinstance(params, torch.Tensor):
        params, grads, momentum_buffers = [params], [grads], [momentum_buffers]
    _refuse_unseen("muon_update", *params, *grads, *momentum_buffers)
    if not (len(params) == len(grads) == len(momentum_buffers)):
        raise NrfError(f"muon_update: {len(params)} parameters, {len(grads)} gradients, {len(momentum_buffers)} momentum buffers")
    if not params:
        return
    shape, dev = params[0].shape, params[0].device
    if len(shape) not in (2, 3):
        raise NrfError(f"muon_update: expected matrices or batches of matrices, got {tuple(shape)}")
    for name, ts in (("param", params), ("grad", grads), ("momentum", momentum_buffers)):
        for t in ts:
            if not t.is_cuda or t.device != dev or t.dtype != torch.float32 or t.shape != shape:
                raise NrfError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, want float32 {tuple(shape)} on {dev}")
            if name != "grad" and not t.is_contiguous():
                raise NrfError(f"{name}: expected a contiguous tensor (it is updated in place)")
    grads = [g.contiguous() for g in grads]
    if _shared([t.data_ptr() for t in (*params, *momentum_buffers)], [g.data_ptr() for g in grads], 4 * shape.numel()):
        raise NrfError("muon_update: tensors overlap (each parameter and momentum buffer is updated in place)")
    rows, cols = shape[-2:]
    batch = shape[0] if len(shape) == 3 else 1
    a, b, c = coefficients
    per = min(len(params), MAX_TENSORS)
    while per > 1 and lib().nrf_newton_schulz_workspace_bytes(batch * per, rows, cols) < 0:
        per //= 2
    for i in range(0, len(params), per):
        part = [ts[i:i + per] for ts in (params, grads, momentum_buffers)]
        n = len(part[0])
        work, need = _workspace(batch * n, rows, cols, dev)
        arrays = [(C.c_void_p * n)(*[t.data_ptr() for t in ts]) for ts in part]
        with _on(dev):
            check(lib().nrf_muon_update(*arrays, n, batch, rows, cols, grad_scale, clip_value, momentum, int(nesterov), lr,
                                        weight_decay, int(steps), a, b, c, eps, _ptr(work), need, _stream(params[0])),
                  "nrf_muon_update")
    _written((*params, *momentum_buffers))

"""Argument checks of the expert entry points: on the host, before any launch (no GPU)."""
import ctypes as C

import pytest
import torch

from nerf_amd import _lib, expert_ops


def test_sizes_out_of_range():
    L = _lib.lib()
    assert L.nrf_expert_plan_bytes(10, 0) == -1 and L.nrf_expert_plan_bytes(10, 16385) == -1
    assert L.nrf_expert_plan_bytes(-1, 4) == -1 and L.nrf_expert_plan_bytes((1 << 28) + 1, 4) == -1
    assert L.nrf_expert_plan_workspace_bytes(8192, 4) == 0 and L.nrf_expert_plan_workspace_bytes(8193, 4) > 0
    assert L.nrf_expert_linear_backward_workspace_bytes(10, 4, 0, 4, 0) == -1
    assert L.nrf_expert_linear_backward_workspace_bytes(10, 4, 4, 4, 3) == -1
    # 4 + 8 words of counts and offsets, 12 of order, 8 run counts, tables of 2 (10 / 32 + 4 + 1) words each, rounded up to four words
    assert L.nrf_expert_plan_bytes(10, 4) == 4 * (4 + 8 + 12 + 8 + 4 * 12)


def test_entry_points_refuse_on_the_host():
    L = _lib.lib()
    p = C.c_void_p(64)                   # never read: every call below is refused before a launch
    odd = C.c_void_p(65)
    need = L.nrf_expert_plan_bytes(10, 4)
    assert L.nrf_expert_plan(p, 10, 0, p, need, None, 0, None) == -2
    assert L.nrf_expert_plan(None, 10, 4, p, need, None, 0, None) == -1
    assert L.nrf_expert_plan(p, 10, 4, None, need, None, 0, None) == -1
    assert L.nrf_expert_plan(p, 10, 4, p, need - 1, None, 0, None) == -4
    assert L.nrf_expert_plan(p, 9000, 4, p, 1 << 30, None, 0, None) == -1
    assert L.nrf_expert_plan(p, 10, 4, odd, need, None, 0, None) == -5
    assert L.nrf_expert_linear(p, p, None, p, 10, 4, 0, 4, 0, 0, p, None) == -2
    assert L.nrf_expert_linear(p, p, None, p, 10, 4, 4, 65537, 0, 0, p, None) == -2
    assert L.nrf_expert_linear(p, p, None, p, 10, 4, 4, 4, 3, 0, p, None) == -2
    assert L.nrf_expert_linear(p, p, None, p, 10, 4, 4, 4, 0, 2, p, None) == -2
    assert L.nrf_expert_linear(None, p, None, p, 10, 4, 4, 4, 0, 0, p, None) == -1
    assert L.nrf_expert_linear(odd, p, None, p, 10, 4, 4, 4, 1, 0, p, None) == -5
    assert L.nrf_expert_linear(p, p, None, p, 0, 4, 4, 4, 0, 0, p, None) == 0
    assert L.nrf_expert_linear_backward(p, p, p, None, p, 10, 4, 4, 4, 0, 1, p, p, p, None, 0, None) == -1   # relu without y
    assert L.nrf_expert_linear_backward(p, p, p, p, p, 10, 4, 4, 4, 0, 1, p, None, p, None, 0, None) == -1   # bias alone
    assert L.nrf_expert_linear_backward(p, p, p, p, p, 10, 4, 4, 4, 0, 1, None, None, None, None, 0, None) == 0
    rows = 1 << 16
    work = L.nrf_expert_linear_backward_workspace_bytes(rows, 2, 64, 64, 0)
    assert work > 0
    assert L.nrf_expert_linear_backward(p, p, p, p, p, rows, 2, 64, 64, 0, 0, p, p, p, p, work - 1, None) == -4


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.NrfError):
        expert_ops.expert_plan(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(_lib.NrfError):
        expert_ops.expert_linear(torch.zeros(4, 4), torch.zeros(2, 4, 4), None, "plan")

"""Tensors that share memory with what a call writes are refused on the host (no GPU: the pointers below are never read, every
call is refused before a launch)."""
import ctypes as C

import pytest

from nerf_amd import _lib, muon_ops

ABC = (3.4445, -4.7750, 2.0315)
SHAPE = -2
MB = 1 << 20


def at(byte):
    return C.c_void_p(byte)


@pytest.mark.parametrize("shift", [-1, 1])
@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_newton_schulz(shift, dtype, size):
    L = _lib.lib()
    # one element less than the whole tensor apart: the last of one is the first of the other
    out = 16 * MB + shift * (3 * 5 * 7 - 1) * size
    assert L.nrf_newton_schulz(at(16 * MB), at(out), 3, 5, 7, dtype, 5, *ABC, 1e-7, None, 0, None) == SHAPE


def test_muon_update():
    L = _lib.lib()
    size = 2 * 20 * 30 * 4

    def call(params, grads, momentum):
        arrays = [(C.c_void_p * len(ts))(*ts) for ts in (params, grads, momentum)]
        return L.nrf_muon_update(*arrays, len(params), 2, 20, 30, 1.0, 40.0, 0.9, 1, 0.02, 0.0, 5, *ABC, 1e-7, None, 0, None)

    p, q, g, m, n = (MB * i for i in range(1, 6))
    for step in (4, size - 4):
        assert call([p], [p + step], [m]) == SHAPE and call([p], [p - step], [m]) == SHAPE
        assert call([p], [g], [p + step]) == SHAPE and call([p], [g], [g + step]) == SHAPE
        assert call([p, p + step], [g, g], [m, n]) == SHAPE and call([p, q], [g, g], [m, m - step]) == SHAPE
        assert call([p, q], [g, n + step], [m, n]) == SHAPE


def test_expert_linear():
    L = _lib.lib()
    n, E, k, m = 10, 3, 16, 16
    x, w, b, y, plan = (at(MB * i) for i in range(1, 6))
    for out in (MB + n * k * 4 - 4, 2 * MB + E * k * m * 4 - 4, 3 * MB + E * m * 4 - 4, MB - n * m * 4 + 4):
        assert L.nrf_expert_linear(x, w, b, plan, n, E, k, m, 0, 0, at(out), None) == SHAPE


def test_expert_linear_backward():
    L = _lib.lib()
    n, E, k, m = 10, 3, 16, 16
    dy, x, w, y, plan, dx, dw, db = (MB * i for i in range(1, 9))
    need = L.nrf_expert_linear_backward_workspace_bytes(n, E, k, m, 0)

    def call(dx=dx, dw=dw, db=db):
        return L.nrf_expert_linear_backward(at(dy), at(x), at(w), at(y), at(plan), n, E, k, m, 0, 1, at(dx), at(dw), at(db), at(9 * MB), need, None)

    row, last = n * k * 4, E * k * m * 4
    assert call(dx=dy) == SHAPE and call(dx=x) == SHAPE and call(dx=y + row - 4) == SHAPE       # in place of an operand
    assert call(dw=w) == SHAPE and call(dw=dx - last + 4) == SHAPE and call(db=dw + last - 4) == SHAPE


def test_shared_ranges():
    shared = muon_ops._shared
    assert not shared([0, 100], [200, 200, 300], 100)          # side by side; gradients may be one another
    assert shared([0, 99], [200], 100) and shared([0, 100], [199], 100) and shared([0, 100], [1], 100) and shared([50], [50], 100)
    assert not shared([0], [100, 150], 100) and shared([200], [100, 150], 100) and shared([249], [100, 150], 100)
    assert not shared([0, 0], [0], 0)

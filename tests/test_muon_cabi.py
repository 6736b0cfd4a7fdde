"""Argument checks of the orthogonalised update's entry points: on the host, before any launch (no GPU)."""
import ctypes as C

import pytest
import torch

from nerf_amd import _lib, muon_ops

ABC = (3.4445, -4.7750, 2.0315)


def test_sizes():
    L = _lib.lib()
    f = L.nrf_newton_schulz_workspace_bytes
    assert f(4096, 32, 63) == 0 and f(4096, 128, 32) == 0 and f(1, 64, 544) == 0 and f(1, 160, 128) == 0     # in registers or LDS
    assert f(1, 64, 545) > 0 and f(1, 65, 161) > 0 and f(1, 129, 129) > 0
    assert f(1, 0, 4) == -1 and f(1, 4, 65537) == -1 and f(-1, 4, 4) == -1 and f(65536, 200, 200) == -1 and f((1 << 24) + 1, 64, 64) == -1
    assert f((1 << 24) + 1, 4, 4) == -1
    assert f(16, 65536, 65536) > 0 and f(17, 65536, 65536) == -1         # 2^24 tiles
    # two terms of 16 bits for X, X^T, both twice, and for A and Q: no size that 32 bits would cut
    assert f(1, 16512, 65536) >= 16 * 16512 * 65536 + 8 * 16512 ** 2


def test_newton_schulz_refuses_on_the_host():
    L = _lib.lib()
    p, odd = C.c_void_p(64), C.c_void_p(66)          # never read: every call below is refused before a launch
    call = lambda g=p, out=p, batch=1, rows=200, cols=200, dtype=0, steps=5, abc=ABC, eps=1e-7, work=p, size=1 << 40: \
        L.nrf_newton_schulz(g, out, batch, rows, cols, dtype, steps, *abc, eps, work, size, None)   # noqa: E731
    assert call(dtype=3) == -2 and call(steps=17) == -2 and call(steps=-1) == -2 and call(eps=0.0) == -2 and call(rows=0) == -2
    assert call(abc=(4.0, 0.0, 0.0)) == -2 and call(abc=(float("nan"), 0.0, 0.0)) == -2
    assert call(g=None) == -1 and call(out=None) == -1 and call(work=None) == -1
    assert call(size=8) == -4 and call(g=odd) == -5 and call(work=C.c_void_p(72)) == -5
    assert call(batch=0) == 0


def test_muon_update_refuses_on_the_host():
    L = _lib.lib()
    p = C.c_void_p(64)
    arr = (C.c_void_p * 1)(64)
    bad = (C.c_void_p * 1)(66)
    null = (C.c_void_p * 1)(None)

    def call(params=arr, grads=arr, mom=arr, n=1, batch=1, clip=40.0, mu=0.9, steps=5, eps=1e-7, work=p, size=1 << 40):
        return L.nrf_muon_update(params, grads, mom, n, batch, 200, 200, 1.0, clip, mu, 1, 0.02, 0.0, steps, *ABC, eps, work, size, None)

    assert call(n=33) == -2 and call(clip=0.0) == -2 and call(mu=1.0) == -2 and call(mu=float("nan")) == -2 and call(steps=20) == -2
    assert call(params=None) == -1 and call(grads=null) == -1 and call(work=None) == -1
    assert call(size=100) == -4 and call(mom=bad) == -5
    assert call(n=0) == 0 and call(batch=0) == 0
    a, b, c = ((C.c_void_p * 2)(x, y) for x, y in ((64, 128), (192, 256), (320, 384)))
    for params, grads, mom in ((a, b, a), (a, a, c), (a, b, b), ((C.c_void_p * 2)(64, 64), b, c), (a, b, (C.c_void_p * 2)(320, 320)),
                               (a, b, (C.c_void_p * 2)(320, 64))):
        assert call(params=params, grads=grads, mom=mom, n=2) == -2      # a tensor twice


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.NrfError):
        muon_ops.newton_schulz(torch.zeros(4, 4))
    with pytest.raises(_lib.NrfError):
        muon_ops.muon_update(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 4))

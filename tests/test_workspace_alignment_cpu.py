"""Workspaces that would be read and written misaligned are refused before any launch."""

from __future__ import annotations

import ctypes

from lightning_router import _ext

P = ctypes.c_void_p(256)     # aligned addresses that a refused call never reads
ODD = ctypes.c_void_p(260)   # a float's alignment, not a double's
N = None
BIG = ctypes.c_size_t(1 << 30)


def test_balanced_gating():
    lbw = ctypes.c_float(0.01)
    f = _ext.clib().lr_balanced_gating
    assert f(P, N, 100000, 8, 2, lbw, P, P, P, P, ODD, BIG, N) == -1
    assert f(P, N, 100000, 8, 2, lbw, P, P, P, P, P, ctypes.c_size_t(8), N) == -4


def test_adapters():
    lib = _ext.clib()
    assert lib.lr_adapter_add(P, 4, 64, P, 2, P, P, N, 8, 64, P, P, ODD, BIG, N, N) == -1
    assert lib.lr_adapter_swiglu(P, 4, 64, P, 2, P, P, N, P, P, N, 8, 64, P, P, P, ODD, BIG, N,
                                 N) == -1

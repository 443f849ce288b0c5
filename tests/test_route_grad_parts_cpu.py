"""The combine's backward takes either gradient alone."""

from __future__ import annotations

import ctypes

from lightning_router import _ext

P = ctypes.c_void_p(256)   # a non-null, aligned address that the call never reads
N = None


def test_neither_gradient_is_nothing_to_do():
    lib = _ext.clib()
    assert lib.lr_combine_backward(P, P, P, P, P, P, 4, 2, 64, 8, N, N, N) == 0
    assert lib.lr_combine_backward(P, P, P, P, P, P, 4, 2, 12, 8, N, N, N) == -1
    assert lib.lr_combine_backward(N, P, P, P, P, P, 4, 2, 64, 8, N, N, N) == -1

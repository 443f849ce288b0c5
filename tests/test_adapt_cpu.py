"""CPU checks of the router-training and adapter entry points: refusals before any CUDA
call, workspace sizes, bank packing."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lightning_router import _ext
from lightning_router.kernels import adapters as ad
from lightning_router.kernels import routing_grad as rg

P = ctypes.c_void_p(256)   # a non-null, aligned address that a refused call never reads
N = None


def test_ops_are_registered():
    ops = _ext.ops()
    for name in ("balanced_gating", "gate_projection", "dispatch_tokens", "combine_tokens",
                 "adapter_add", "adapter_swiglu", "adapter_rows"):
        assert hasattr(ops, name), name


def test_workspace_sizes():
    lib = _ext.clib()
    f = lib.lr_balanced_gating_workspace_bytes
    assert f(0, 8) == 0 and f(512, 8) == 0      # one block: no partials
    assert f(513, 8) >= 2 * (8 * 8 + 9 * 4)     # two blocks: sums and counts
    assert f(1 << 24, 64) == f(1 << 20, 64)     # a bounded grid
    g = lib.lr_gate_backward_workspace_bytes
    # two fp16 terms per gradient, the transposed weight, partial sums once there are ranges
    assert g(0, 4096, 8) == 0 and g(256, 4096, 64) == 0      # small batches need none
    assert g(257, 4096, 8) >= 257 * 8 * 4 + 4096 * 8 * 2 and g(16, 4096, 65) > 0
    assert g(16384, 4096, 8) >= 16384 * 8 * 4 + 4096 * 8 * 2 + 2 * 4096 * 8 * 4
    h = lib.lr_adapter_workspace_bytes
    assert h(64, 16, 1) == 64 * 16 * 4 and h(64, 16, 2) == 2 * h(64, 16, 1) and h(0, 16, 1) == 0


def test_gating_arguments():
    lib = _ext.clib()
    lbw, ws = ctypes.c_float(0.01), ctypes.c_size_t(0)
    for T, E, k in [(-1, 8, 2), (4, 0, 1), (4, 65, 2), (4, 8, 0), (4, 4, 5), (4, 64, 9)]:
        assert lib.lr_balanced_gating(P, N, T, E, k, lbw, P, P, P, P, N, ws, N) == -1
        assert lib.lr_balanced_gating_backward(P, N, P, P, 0, P, P, T, E, k, lbw, P, N) == -1
    assert lib.lr_balanced_gating(P, N, 4, 8, 2, lbw, P, P, N, P, N, ws, N) == -1
    assert lib.lr_balanced_gating(P, N, 4096, 8, 2, lbw, P, P, P, P, N, ws, N) == -4
    # a mask does not go with a dispatch's offsets; nothing to do for no tokens
    assert lib.lr_balanced_gating_backward(P, P, P, P, 1, P, P, 4, 8, 2, lbw, P, N) == -1
    assert lib.lr_balanced_gating_backward(N, N, N, N, 0, N, N, 0, 8, 2, lbw, N, N) == 0


def test_gradient_arguments():
    lib = _ext.clib()
    ws = ctypes.c_size_t(0)
    for T, d, E in [(-1, 64, 8), (4, 24, 8), (4, 0, 8), (4, 64, 0), (4, 64, 257)]:
        assert lib.lr_gate_backward(P, P, P, T, d, E, P, P, P, N, ws, N) == -1
    assert lib.lr_gate_backward(P, P, P, 4, 64, 8, P, N, P, N, ws, N) == -1   # bias without weight
    assert lib.lr_gate_backward(ctypes.c_void_p(258), P, P, 4, 64, 8, P, P, N, N, ws, N) == -1
    assert lib.lr_gate_backward(P, P, P, 16384, 4096, 8, N, P, N, N, ws, N) == -4
    for T, k, d in [(-1, 2, 64), (4, 0, 64), (4, 9, 64), (4, 2, 12)]:
        assert lib.lr_dispatch_backward(P, P, T, k, d, P, N) == -1
        assert lib.lr_combine_backward(P, P, P, P, P, P, T, k, d, 8, P, P, N) == -1
    assert lib.lr_combine_backward(P, P, N, P, P, P, 4, 2, 64, 8, P, P, N) == -1
    assert lib.lr_dispatch_backward(N, N, 0, 2, 64, N, N) == 0


def test_round_half_arguments():
    lib = _ext.clib()
    n = ctypes.c_longlong
    assert lib.lr_round_half(P, P, n(12), N) == -1 and lib.lr_round_half(P, P, n(-8), N) == -1
    assert lib.lr_round_half(ctypes.c_void_p(260), P, n(8), N) == -1
    assert lib.lr_round_half(N, N, n(0), N) == 0


def test_adapter_arguments():
    lib = _ext.clib()
    big = ctypes.c_size_t(1 << 20)
    for R, K, n, r, F in [(-1, 64, 2, 8, 64), (4, 60, 2, 8, 64), (4, 64, 0, 8, 64),
                          (4, 64, 2, 4, 64), (4, 64, 2, 12, 64), (4, 64, 2, 136, 64),
                          (4, 64, 2, 8, 60), (4, 0, 2, 8, 64)]:
        assert lib.lr_adapter_add(P, R, K, P, n, P, P, N, r, F, P, P, P, big, N, N) == -1
        assert lib.lr_adapter_swiglu(P, R, K, P, n, P, P, N, P, P, N, r, F, P, P, P, P, big, N,
                                     N) == -1
    assert lib.lr_adapter_add(P, 4, 64, N, 2, P, P, N, 8, 64, P, P, P, big, N, N) == -1
    assert lib.lr_adapter_add(ctypes.c_void_p(264), 4, 64, P, 2, P, P, N, 8, 64, P, P, P, big, N,
                              N) == -1
    small = ctypes.c_size_t(4 * 8 * 4 - 1)
    assert lib.lr_adapter_add(P, 4, 64, P, 2, P, P, N, 8, 64, P, P, P, small, N, N) == -4
    assert lib.lr_adapter_add(N, 0, 64, N, 2, N, N, N, 8, 64, N, N, N, big, N, N) == 0
    assert lib.lr_adapter_rows(P, 4, 0, P, P, P, 8, 4, P, N, N) == -1
    assert lib.lr_adapter_rows(P, 4, 1 << 30, P, P, P, 8, 4, P, N, N) == -1


def test_sizes_past_32_bit_offsets_are_refused():
    lib = _ext.clib()
    lbw, ws, big = ctypes.c_float(0.01), ctypes.c_size_t(0), ctypes.c_size_t(1 << 62)
    top = 2**31 - 1
    assert lib.lr_balanced_gating(P, N, top, 8, 2, lbw, P, P, P, P, P, big, N) == -1
    assert lib.lr_balanced_gating_backward(P, N, P, P, 0, P, P, top, 8, 2, lbw, P, N) == -1
    assert lib.lr_gate_backward(P, P, P, top, 64, 8, P, P, N, P, big, N) == -1
    assert lib.lr_gate_backward(P, P, P, 4, (1 << 26) + 16, 8, P, P, N, N, ws, N) == -1
    assert lib.lr_dispatch_backward(P, P, 1 << 29, 4, 64, P, N) == -1
    assert lib.lr_combine_backward(P, P, P, P, P, P, 1 << 29, 4, 64, 8, P, P, N) == -1
    for R, K, F in [(top, 64, 64), (64, (1 << 26) + 8, 64), (64, 64, (1 << 26) + 8)]:
        assert lib.lr_adapter_add(P, R, K, P, 2, P, P, N, 8, F, P, P, P, big, N, N) == -1
    assert lib.lr_adapter_rows(P, 4, 2, P, P, P, top, 4, P, N, N) == -1


def test_adapters_of_another_layer_are_refused():
    from lightning_router.models.adapters import ExpertAdapters
    from lightning_router.models.experts import ExpertGroup
    swiglu = ExpertGroup(4, 64, 128, quantized=True, group_size=64)
    silu = ExpertGroup(4, 64, 128, quantized=True, group_size=64, activation="silu")
    ExpertAdapters(2, 4, 64, 128, 8).check(swiglu)
    ExpertAdapters(2, 4, 64, 128, 8, gated=False).check(silu)
    for other, experts in [(ExpertAdapters(2, 8, 64, 128, 8), swiglu),
                           (ExpertAdapters(2, 4, 128, 128, 8), swiglu),
                           (ExpertAdapters(2, 4, 64, 64, 8), swiglu),
                           (ExpertAdapters(2, 4, 64, 128, 8, gated=False), swiglu),
                           (ExpertAdapters(2, 4, 64, 128, 8), silu)]:
        with pytest.raises(RuntimeError, match="adapters for"):
            other.check(experts)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        rg.balanced_gating(x, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        rg.gate_projection(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        rg.dispatch_tokens(x, x, 2)
    bank = ad.pack_adapters([(torch.zeros(8, 16), torch.zeros(16, 8))])
    with pytest.raises(RuntimeError, match="CUDA"):
        ad.adapter_add(x.half(), x.half(), bank, torch.zeros(4, dtype=torch.int32))


def test_pack_adapters():
    pairs = [(torch.full((r, 24), float(r)), torch.full((16, r), -float(r))) for r in (3, 9)]
    bank = ad.pack_adapters(pairs, [0.5, 2.0])
    assert bank.a.shape == (2, 16, 24) and bank.b.shape == (2, 16, 16)
    assert bank.a.dtype == bank.b.dtype == torch.float16 and bank.scale.tolist() == [0.5, 2.0]
    assert bool((bank.a[0, :3] == 3).all()) and not bank.a[0, 3:].any()
    assert bool((bank.b[1, :, :9] == -9).all()) and not bank.b[1, :, 9:].any()
    assert ad.pack_adapters(pairs).scale is None
    with pytest.raises(ValueError, match="no adapters"):
        ad.pack_adapters([])
    with pytest.raises(ValueError, match="scales"):
        ad.pack_adapters(pairs, [1.0])
    with pytest.raises(ValueError, match="expected"):
        ad.pack_adapters([(torch.zeros(4, 8), torch.zeros(16, 5))])

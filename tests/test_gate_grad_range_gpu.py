"""The gate projection's gradients over fp32's range of logit gradients, the same on both sides of
the switch between the one-launch form and the split fp16 products (256 tokens, 64 experts).

Tolerances as in the gate projection's own test: 4 U per step of a tensor-core sum times the
terms' magnitudes (``U = 2^-24``) and, for the row gradient, 2^-22 of a row's largest; terms or
remainders below the normal range lose at most 2^-126 of the weight or row they multiply."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.parametrize("T,E", [(200, 8), (256, 64), (257, 8), (257, 64), (3000, 33), (700, 100)])
@pytest.mark.parametrize("size", [1e-33, 1e-20, 1e20, 1e34, 3e35])
def test_small_and_large_logit_gradients(T, E, size):
    from lightning_router.kernels.routing_grad import gate_projection
    g = torch.Generator(device=DEV).manual_seed(T + E)
    h = torch.randn(T, 128, generator=g, device=DEV).half().float().requires_grad_()
    w = (torch.randn(E, 128, generator=g, device=DEV) * 0.05).half().float().requires_grad_()
    dl = (torch.randn(T, E, generator=g, device=DEV).double() * size).float()
    dh, dw = torch.autograd.grad(gate_projection(h, w), (h, w), dl)
    d64, h64, w64 = dl.double(), h.detach().double(), w.detach().double()
    want = d64.t() @ h64
    tol = (64 + 8 + T // 128 + 8) * 4 * U * (d64.abs().t() @ h64.abs()) \
        + 2.0 ** -126 * h64.abs().sum(0)
    assert want.abs().max() < 3e38
    assert bool(((dw.double() - want).abs() <= tol).all())
    want = d64 @ w64
    tol = (E // 4 + 8) * 4 * U * (d64.abs() @ w64.abs()) + U * want.abs() \
        + (2.0 ** -22 * d64.abs().amax(1, keepdim=True) + 2.0 ** -126) * w64.abs().sum(0)
    assert bool(((dh.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("T", [200, 300])
def test_a_column_of_mixed_sizes(T):
    """One huge gradient among ordinary ones of an expert: finite where the sums are."""
    from lightning_router.kernels.routing_grad import gate_projection
    g = torch.Generator(device=DEV).manual_seed(T)
    h = torch.randn(T, 64, generator=g, device=DEV).requires_grad_()
    w = torch.randn(5, 64, generator=g, device=DEV).requires_grad_()
    dl = torch.randn(T, 5, generator=g, device=DEV)
    dl[3, 2], dl[4, 1] = 3e37, -1e38
    dh, dw = torch.autograd.grad(gate_projection(h, w), (h, w), dl)
    d64, h64 = dl.double(), h.detach().half().double()
    want = d64.t() @ h64
    keep = want.abs() < 2.0 ** 127
    tol = (64 + 8 + T // 128 + 8) * 4 * U * (d64.abs().t() @ h64.abs())
    assert bool(((dw.double() - want).abs() <= tol)[keep].all())
    assert bool(torch.isfinite(dw[[0, 3, 4]]).all())
    w64 = w.detach().half().double()
    want = d64 @ w64
    keep = want.abs() < 2.0 ** 127
    tol = 9 * 4 * U * (d64.abs() @ w64.abs()) + U * want.abs() \
        + 2.0 ** -22 * d64.abs().amax(1, keepdim=True) * w64.abs().sum(0)
    assert bool(((dh.double() - want).abs() <= tol)[keep].all())

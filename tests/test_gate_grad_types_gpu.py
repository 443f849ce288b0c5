"""The gate projection's gradients for hidden rows of every type, from tiny to huge.

A row gradient is a sum of E products ``dl W`` in fp32 (off by at most 4 U times the terms'
magnitudes per step of a tensor-core sum, ``U = 2^-24``), in the large batches with ``dl`` in two
fp16 or tf32 terms (2^-22 of its row's largest left over), rounded once to the hidden rows' type
(half a step: 2^-8 of the value for bf16, 2^-24 for fp32).  There is no absolute term: a gradient
far below or above fp16's range keeps its relative precision.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24

# both sides of the one-launch form (256 tokens, 64 experts), of 16, 32, 64 and 128 experts, of
# the low-rank product's window sizes
SHAPES = [(1, 16, 1), (100, 64, 7), (256, 496, 64), (257, 496, 64), (100, 64, 65), (300, 1040, 8),
          (1000, 512, 33), (3001, 2000, 100), (9000, 2048, 16), (300, 64, 130), (777, 4096, 129)]


@pytest.mark.parametrize("T,d,E", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("size", [1e-9, 1.0, 1e8])
def test_row_gradients_keep_the_hidden_type(T, d, E, dtype, size):
    from lightning_router.kernels.routing_grad import gate_projection
    g = torch.Generator(device=DEV).manual_seed(T + d + E)
    h = torch.randn(T, d, generator=g, device=DEV).to(dtype).requires_grad_()
    w = (torch.randn(E, d, generator=g, device=DEV) * 0.05).requires_grad_()
    dl = torch.randn(T, E, generator=g, device=DEV) * size
    out = gate_projection(h, w)
    assert torch.equal(out.detach(), gate_projection(h.detach().half(), w.detach()))
    dh, dw = torch.autograd.grad(out, (h, w), dl)
    assert dh.dtype == dtype and dw.dtype == torch.float32
    w64, d64 = w.detach().half().double(), dl.double()
    want = d64 @ w64
    tol = (E // 4 + 8) * 4 * U * (d64.abs() @ w64.abs()) \
        + 2.0 ** -22 * d64.abs().amax(1, keepdim=True) * w64.abs().sum(0)
    tol = tol + want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else U)
    err = (dh.double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()))
    h64 = h.detach().half().double()
    tol = (64 + 8 + T // 128 + 8) * 4 * U * (d64.abs().t() @ h64.abs())
    assert bool(((dw.double() - d64.t() @ h64).abs() <= tol).all())


@pytest.mark.parametrize("T,E", [(50, 8), (700, 40), (700, 140)])
def test_fp16_rows_get_the_same_sums_rounded(T, E):
    """One set of sums: the fp16 gradient is the fp32 one's rounding."""
    from lightning_router.kernels.routing_grad import gate_projection
    g = torch.Generator(device=DEV).manual_seed(E)
    h = torch.randn(T, 256, generator=g, device=DEV).half()
    w = torch.randn(E, 256, generator=g, device=DEV)
    dl = torch.randn(T, E, generator=g, device=DEV)
    grads = {}
    for dtype in (torch.float16, torch.float32):
        leaf = h.to(dtype).requires_grad_()
        (grads[dtype],) = torch.autograd.grad(gate_projection(leaf, w), leaf, dl)
    assert torch.equal(grads[torch.float16], grads[torch.float32].half())


def test_trainable_gate_module_with_small_gradients():
    """A loss averaged over tokens, unscaled, and fp32 hidden states."""
    from lightning_router.models.gating import TopKGating
    torch.manual_seed(1)
    gate = TopKGating(256, 16, 2, load_balance_weight=1e-4, trainable=True).to(DEV)
    x = torch.randn(4000, 256, device=DEV, requires_grad=True)
    aux = gate(x)[3]
    (small,) = torch.autograd.grad(aux, x)
    (large,) = torch.autograd.grad(gate(x)[3] * 2.0 ** 20, x)
    assert small.abs().max() < 2.0 ** -24       # below fp16's smallest
    assert torch.equal(small * 2.0 ** 20, large)

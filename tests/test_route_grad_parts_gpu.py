"""Gradients of dispatch and combine that nobody asks for are neither computed nor allocated, and
the others keep their bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(T, d, E, k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=DEV)
    return (randn(T, d).half(), randn(T, E), randn(T * k, d).half(), randn(T, d).half(),
            randn(T * k, d).half())


@pytest.mark.parametrize("T,d,E,k,cf", [(1, 8, 2, 1, 1.25), (300, 520, 8, 2, 0.7),
                                        (700, 64, 64, 8, 0.1), (3000, 264, 4, 2, 1.0)])
def test_parts_keep_their_bits(T, d, E, k, cf):
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    x, logits, y, dout, dperm = _case(T, d, E, k, T + d)
    w0 = dispatch_tokens(x, logits, k, cf).gate_weights

    def grads(**need):
        xl, ll, yl, wl = (t.clone().requires_grad_(need.get(n, False))
                          for n, t in zip("xlyw", (x, logits, y, w0)))
        plan = dispatch_tokens(xl, ll, k, cf)
        out = combine_tokens(yl, wl, plan)
        outs, gs = [], []
        if need.get("y") or need.get("w"):
            outs.append(out), gs.append(dout)
        if need.get("x") or need.get("l"):
            outs += [plan.permuted, plan.gate_weights, plan.aux_loss]
            gs += [dperm, w0, torch.ones((), device=DEV)]
        torch.autograd.backward(outs, gs)
        return dict(x=xl.grad, l=ll.grad, y=yl.grad, w=wl.grad)

    full = grads(x=True, l=True, y=True, w=True)
    for n in "xlyw":
        part = grads(**{n: True})
        assert torch.equal(part[n], full[n]), n
        assert all(part[m] is None for m in "xlyw" if m != n)


def test_inputs_named_to_autograd():
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    x, logits, y, dout, _ = _case(200, 64, 4, 2, 5)
    plan = dispatch_tokens(x, logits, 2)
    yl, wl = y.clone().requires_grad_(), plan.gate_weights.clone().requires_grad_()
    out = combine_tokens(yl, wl, plan)
    dy, dw = torch.autograd.grad(out, (yl, wl), dout, retain_graph=True)
    (a,) = torch.autograd.grad(out, yl, dout, retain_graph=True)
    (b,) = torch.autograd.grad(out, wl, dout)
    assert torch.equal(a, dy) and torch.equal(b, dw)


def test_frozen_rows_cost_no_memory():
    """A router over frozen experts: T k d fp16 values that nobody reads were written."""
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    T, d, k = 4096, 2048, 2
    x, logits, y, dout, _ = _case(T, d, 8, k, 1)
    leaf = logits.clone().requires_grad_()
    plan = dispatch_tokens(x, leaf, k)
    out = combine_tokens(y, plan.gate_weights, plan)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out.backward(dout)
    assert leaf.grad is not None
    assert torch.cuda.max_memory_allocated() - before < T * k * d

"""Adapters written into a given tensor are an in-place change that autograd sees."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(R=64, K=64, N=64, n=3, r=8, seed=0):
    from lightning_router.kernels.adapters import AdapterBank
    g = torch.Generator(device=DEV).manual_seed(seed)

    def half(*s):
        return torch.randn(*s, generator=g, device=DEV).half()
    bank = AdapterBank(half(n, r, K), half(n, N, r))
    ids = torch.randint(-1, n, (R,), generator=g, device=DEV, dtype=torch.int32)
    return half(R, K), half(R, N), half(R, N), bank, ids


def _write(op, y, x, up, bank, ids):
    from lightning_router.kernels.adapters import adapter_add, adapter_swiglu
    if op == "add":
        return adapter_add(y, x, bank, ids, out=y)
    return adapter_swiglu(y, up, x, bank, bank, ids, out=y)


@pytest.mark.parametrize("op", ["add", "swiglu"])
def test_rows_saved_for_a_gradient_and_overwritten(op):
    """combine saves the experts' rows for its weights' gradient."""
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    x, y, up, bank, ids = _case(R=64)
    logits = torch.randn(32, 4, device=DEV)
    plan = dispatch_tokens(x[:32], logits, 2)
    w = plan.gate_weights.detach().requires_grad_()
    out = combine_tokens(y, w, plan)
    assert _write(op, y, x, up, bank, ids) is y
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()


@pytest.mark.parametrize("op", ["add", "swiglu"])
def test_hidden_rows_saved_by_the_gate_and_overwritten(op):
    from lightning_router.kernels.routing_grad import gate_projection
    x, y, up, bank, ids = _case()
    w = torch.randn(4, 64, device=DEV, requires_grad=True)
    out = gate_projection(y, w)
    _write(op, y, x, up, bank, ids)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("op", ["add", "swiglu"])
def test_a_leaf_is_not_overwritten(op):
    from lightning_router.kernels.adapters import adapter_add, adapter_swiglu
    x, y, up, bank, ids = _case()
    leaf = torch.zeros_like(y).requires_grad_()

    def call():
        if op == "add":
            return adapter_add(y, x, bank, ids, out=leaf)
        return adapter_swiglu(y, up, x, bank, bank, ids, out=leaf)
    with pytest.raises(RuntimeError, match="no backward"):
        call()
    assert not leaf.detach().any()
    before = leaf._version
    with torch.no_grad():
        assert call() is leaf and leaf._version == before + 1 and leaf.requires_grad


def test_without_out_nothing_given_changes():
    from lightning_router.kernels.adapters import adapter_add
    x, y, _, bank, ids = _case()
    versions = [t._version for t in (x, y, bank.a, bank.b, ids)]
    a = adapter_add(y, x, bank, ids)
    assert [t._version for t in (x, y, bank.a, bank.b, ids)] == versions
    assert torch.equal(adapter_add(y.clone(), x, bank, ids, out=y), a)


def test_inference_tensors_are_written_as_before():
    from lightning_router.kernels.adapters import adapter_add
    x, y, _, bank, ids = _case()
    want = adapter_add(y, x, bank, ids)
    with torch.inference_mode():
        z = y.clone()
        assert torch.equal(adapter_add(z, x, bank, ids, out=z), want)
    with torch.inference_mode():
        z = y.clone()
    assert torch.equal(adapter_add(z, x, bank, ids, out=z), want)

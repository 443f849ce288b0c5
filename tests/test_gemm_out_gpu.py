"""Expert products written into a given tensor are an in-place change that autograd sees."""

from __future__ import annotations

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_expert_rows_saved_for_a_gradient_and_overwritten():
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    from lightning_router.workloads import WORKLOADS, build_layer
    layer, t = build_layer(dataclasses.replace(WORKLOADS["decode"], tokens=32, d_model=256,
                                               d_ff=256), device=DEV)
    with torch.no_grad():
        logits = layer.gate.logits(t.x)
        plan = dispatch_tokens(t.x, logits, layer.top_k, capacity=layer.capacity(32))
        y = layer.expert_forward(plan)
    for again in (False, True):
        w = plan.gate_weights.detach().requires_grad_()
        out = combine_tokens(y, w, plan)
        before = y._version
        if again:
            same = layer.experts.forward_segments(plan.permuted, plan.offsets[:-1],
                                                  plan.kept_counts, plan.capacity, out=y)
            assert same.data_ptr() == y.data_ptr() and y._version > before
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.float().sum().backward()
        else:
            out.float().sum().backward()
            assert w.grad.abs().sum() > 0


def test_a_given_result_in_inference_mode():
    from lightning_router.workloads import WORKLOADS, build_layer
    layer, t = build_layer(dataclasses.replace(WORKLOADS["decode"], tokens=16, d_model=256,
                                               d_ff=256), device=DEV)
    with torch.inference_mode():
        _, plan = layer.route(t.x)
        args = (plan.permuted, plan.offsets[:-1], plan.kept_counts, plan.capacity)
        y = torch.zeros(plan.permuted.shape[0], 256, dtype=torch.float16, device=DEV)
        layer.experts.forward_segments(*args, out=y)
        want = layer.experts.forward_segments(*args)
    kept = plan.kept_counts.tolist()
    off = plan.offsets.tolist()
    for e, n in enumerate(kept):
        assert torch.equal(y[off[e]:off[e] + n], want[off[e]:off[e] + n])

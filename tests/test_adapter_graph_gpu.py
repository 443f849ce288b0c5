"""A captured step with adapters is replayed only while they are where the graph reads them."""

from __future__ import annotations

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _runner(tokens=16, d=256, f=512, E=8, n=4, rank=8):
    from lightning_router.models.adapters import ExpertAdapters
    from lightning_router.serving.model_runner import LightningModelRunner
    from lightning_router.workloads import WORKLOADS, build_layer
    layer, _ = build_layer(dataclasses.replace(WORKLOADS["decode"], tokens=tokens, d_model=d,
                                               d_ff=f), device=DEV)
    r = LightningModelRunner(dict(hidden_size=d, intermediate_size=f),
                             dict(num_experts=E, num_experts_per_token=2), dict(group_size=128),
                             {}, device="cuda:0")
    r.load_model()
    r.moe_layer.load_state_dict(layer.state_dict())
    g = torch.Generator(device=DEV).manual_seed(3)
    ad = ExpertAdapters(n, E, d, f, rank).to(DEV)
    for m in ad.mats:
        for part, std in (("a", 0.06), ("b", 0.05)):
            t = getattr(ad, f"{m}_{part}")
            t.copy_(torch.randn(t.shape, generator=g, device=DEV) * std)
    r.set_adapters(ad)
    r.capture(tokens, adapters=True)
    x = torch.randn(tokens, d, generator=g, device=DEV).half()
    ids = torch.arange(tokens, device=DEV, dtype=torch.int32) % n
    return r, ad, x, ids


def _replayed(r):
    """Counts the replays of the captured graphs."""
    seen = []
    for gr in r._graphs.values():
        class Counted:
            def __init__(self, graph):
                self.graph = graph

            def replay(self):
                seen.append(1)
                self.graph.replay()
        gr.graph = Counted(gr.graph)
    return seen


def _check(r, x, ids):
    ref, _ = r.moe_layer(x, adapter_ids=ids)
    assert torch.equal(r.execute_model(None, x, adapter_ids=ids), ref)
    return ref


def test_values_changed_in_place_are_replayed():
    r, ad, x, ids = _runner()
    seen = _replayed(r)
    old = _check(r, x, ids)
    ad.up_b.mul_(2)
    ad.load(1, 3, "down", torch.randn(8, 512, device=DEV), torch.randn(256, 8, device=DEV), 0.5)
    assert not torch.equal(_check(r, x, ids), old) and len(seen) == 2


@pytest.mark.parametrize("how", ["assigned", "data", "state", "moved", "half"])
def test_buffers_replaced(how):
    r, ad, x, ids = _runner()
    seen = _replayed(r)
    old = _check(r, x, ids)
    assert len(seen) == 1
    if how == "assigned":
        ad.up_a = ad.up_a * 3
    elif how == "data":
        ad.up_a.data = ad.up_a * 3
    elif how == "state":
        ad.load_state_dict({k: v * 3 for k, v in ad.state_dict().items()}, assign=True)
    elif how == "moved":
        ad.cpu()
        ad.to(DEV)
        ad.up_a.mul_(3)
    else:
        ad.double()
        ad.half()            # new memory for the same values, the scales fp16 now
        ad.up_a.mul_(3)
    torch.cuda.empty_cache()
    filler = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(4)]
    new = _check(r, x, ids)
    assert len(seen) == 1 and not torch.equal(new, old)      # eager, with the new values
    r.capture(16, adapters=True)
    seen = _replayed(r)
    assert torch.equal(_check(r, x, ids), new) and len(seen) == 1
    del filler

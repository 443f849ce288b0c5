"""When a captured step with adapters may be replayed, with a stand-in for graph and layer."""

from __future__ import annotations

import pytest
import torch

from lightning_router.models.adapters import ExpertAdapters
from lightning_router.serving.model_runner import LightningModelRunner, _Graph


class _Layer:
    def __init__(self, adapters):
        self.adapters = adapters

    def __call__(self, h, adapter_ids=None):
        return torch.full_like(h, 2.0), None


class _Replay:
    def __init__(self):
        self.n = 0

    def replay(self):
        self.n += 1


def _runner():
    ad = ExpertAdapters(2, 3, 16, 24, 8)
    r = LightningModelRunner({}, {}, {}, {}, device="cpu")
    r.moe_layer = _Layer(ad)
    x, ids, replay = torch.zeros(4, 16), torch.zeros(4, dtype=torch.int32), _Replay()
    r._graphs[(4, 16, True)] = _Graph(replay, torch.empty(4, 16), torch.ones(4, 16), None, ids, ad)
    return r, ad, x, ids, replay


def test_the_same_memory_is_replayed():
    r, ad, x, ids, replay = _runner()
    assert r.execute_model(None, x, adapter_ids=ids).eq(1).all() and replay.n == 1
    ad.load(1, 2, "up", torch.ones(5, 16), torch.ones(24, 5))      # in place
    assert r.execute_model(None, x, adapter_ids=ids).eq(1).all() and replay.n == 2


@pytest.mark.parametrize("how", ["assigned", "data", "state", "types", "module", "none"])
def test_other_memory_is_not(how):
    r, ad, x, ids, replay = _runner()
    if how == "assigned":
        ad.down_scale = ad.down_scale.clone()
    elif how == "data":
        ad.gate_b.data = ad.gate_b.clone()
    elif how == "state":
        ad.load_state_dict({k: v.clone() for k, v in ad.state_dict().items()}, assign=True)
    elif how == "types":
        ad.double()
        ad.half()
    elif how == "module":
        r.moe_layer.adapters = ExpertAdapters(2, 3, 16, 24, 8)
    else:
        r.moe_layer.adapters = None
    assert r.execute_model(None, x, adapter_ids=ids).eq(2).all() and replay.n == 0


def test_the_captured_memory_is_kept():
    r, ad, x, ids, replay = _runner()
    gr = r._graphs[(4, 16, True)]
    at = ad.up_a.data_ptr()
    ad.up_a = ad.up_a.clone()
    assert any(b.data_ptr() == at for b in gr.banks)

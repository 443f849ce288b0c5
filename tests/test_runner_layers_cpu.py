"""The runner calls a layer that knows no adapters as it always did."""

from __future__ import annotations

import pytest
import torch

from lightning_router.serving.model_runner import LightningModelRunner


class _Plain(torch.nn.Module):
    def forward(self, h):
        return h * 2, torch.zeros(())


def test_a_layer_without_adapter_ids():
    r = LightningModelRunner({}, {}, {}, {}, device="cpu")
    r.moe_layer = _Plain()
    x = torch.ones(2, 3, 8)
    assert torch.equal(r.execute_model(None, x), x * 2)
    with pytest.raises(TypeError):
        r.execute_model(None, x, adapter_ids=torch.zeros(6, dtype=torch.int32))

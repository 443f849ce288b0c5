"""The route kernel's two forms (a thread per token, several lanes per token) give the same bits:
a batch large enough for the first against its tokens in batches small enough for the second."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T,E,k", [(40001, 24, 4), (76033, 16, 2), (20000, 32, 8), (50500, 12, 3),
                                   (76033, 9, 2)])
def test_large_route_is_the_small_ones_bit_for_bit(T, E, k):
    from lightning_router.kernels.expert_routing import topk_gating_dispatch
    g = torch.Generator(device=DEV).manual_seed(T + E)
    logits = torch.randn(T, E, generator=g, device=DEV)
    logits[::97, ::2] = logits[::97, :1]                  # ties
    logits[5::1001, 1] = float("nan")                     # a NaN that is passed over
    logits[6::1001, 0] = float("nan")                     # and one that is selected
    logits[7::1001, 1::2] = float("-inf")
    big = topk_gating_dispatch(None, logits, k)
    part = 128 * 20
    counts = torch.zeros(E, dtype=torch.int64, device=DEV)
    for lo in range(0, T, part):
        p = topk_gating_dispatch(None, logits[lo:lo + part], k)
        s = slice(lo * k, min(lo + part, T) * k)
        assert torch.equal(big.expert_ids[s], p.expert_ids)
        assert torch.equal(big.gate_weights[s].view(torch.int32), p.gate_weights.view(torch.int32))
        counts += p.offsets.diff()
    # slots per expert, and each slot's place among its expert's
    assert torch.equal(big.offsets.diff().long(), counts)
    assert torch.equal(torch.bincount(big.expert_ids.long(), minlength=E), counts)

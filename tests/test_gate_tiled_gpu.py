"""Gate logits of large batches: the tiled kernel against the small-batch kernel, bit for bit
(rows of the same token in batches below and above the switch between them)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2048, 2049, 2111])
@pytest.mark.parametrize("d,E", [(16, 1), (64, 8), (144, 5), (1024, 9), (2048, 64), (4096, 8),
                                 (400, 33), (256, 130), (1040, 17), (96, 256)])
@pytest.mark.parametrize("bias", [False, True])
def test_tiled_logits_are_the_same_bits(T, d, E, bias):
    from lightning_router.kernels.expert_routing import gate_logits
    g = torch.Generator(device="cuda").manual_seed(d + E)
    h = torch.randn(T, d, generator=g, device="cuda").half()
    w = (torch.randn(E, d, generator=g, device="cuda") * 0.05).half()
    b = torch.randn(E, generator=g, device="cuda") if bias else None
    big = gate_logits(h, w, b)
    for lo in range(0, T, 1000):
        assert torch.equal(big[lo:lo + 1000], gate_logits(h[lo:lo + 1000], w, b))

"""Gate logits on both sides of every switch between the tiled and the untiled kernel: the same
bits as the same rows in batches below 2048 tokens, which are never tiled."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,d,E", [
    (9471, 64, 8), (9472, 64, 8), (9473, 16, 1), (9500, 144, 16), (9472, 240, 5),   # short rows
    (2048, 240, 8), (2048, 256, 8), (4095, 496, 32), (4095, 512, 32), (2050, 1008, 64),
    (2050, 1024, 33), (4095, 256, 64), (4096, 256, 64), (4097, 240, 64), (4096, 272, 17),
    (2048, 240, 130), (2048, 256, 130)])
def test_logits_at_the_switches(T, d, E):
    from lightning_router.kernels.expert_routing import gate_logits
    g = torch.Generator(device="cuda").manual_seed(T + d + E)
    h = torch.randn(T, d, generator=g, device="cuda").half()
    w = (torch.randn(E, d, generator=g, device="cuda") * 0.05).half()
    b = torch.randn(E, generator=g, device="cuda")
    big = gate_logits(h, w, b)
    for lo in range(0, T, 2000):
        assert torch.equal(big[lo:lo + 2000], gate_logits(h[lo:lo + 2000], w, b))

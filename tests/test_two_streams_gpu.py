"""Two steps of a layer at once, each on a stream of its own: the bits of one alone.

Blocks of one step then start beside the other step's, and copies land in other orders than in a
quiet GPU."""

from __future__ import annotations

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("name,kw,rounds", [
    ("prefill", dict(tokens=8192, d_ff=4096), 40),        # 256-row tiles, 3 stages, 2 groups
    ("decode", dict(tokens=256, d_ff=4096), 100),         # 64- and 128-row tiles
    ("decode", dict(tokens=64, d_ff=4096), 100),
    ("fine", dict(tokens=3000), 60)])
def test_concurrent_layers(name, kw, rounds):
    from lightning_router import _ext
    from lightning_router.workloads import WORKLOADS, build_layer
    layer, t = build_layer(dataclasses.replace(WORKLOADS[name], **kw), device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    xs = [torch.randn(t.x.shape, generator=g, device=DEV).half() for _ in range(3)]
    want = []
    for x in xs:
        want.append(layer(x)[0])
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(rounds):
        got = []
        for n, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(layer(xs[(i + n) % 3])[0])
        torch.cuda.synchronize()
        for n, o in enumerate(got):
            assert torch.equal(o, want[(i + n) % 3]), (i, n)
    _ext.check_device_errors()


@pytest.mark.parametrize("M", [33, 64, 65, 128, 129, 600])
def test_concurrent_products(M):
    from lightning_router.kernels.quantized_matmul import quantized_matmul
    from lightning_router.quantization.pack_weights import quantize_tensor
    K, N = 4096, 2048
    g = torch.Generator().manual_seed(M)
    q, s, z = (v.to(DEV) for v in quantize_tensor(torch.randn(K, N, generator=g) * 0.02, 128))
    xs = [torch.randn(M, K, generator=g).half().to(DEV) for _ in range(3)]
    want = []
    for x in xs:
        want.append(quantized_matmul(x, q, s, z, N))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(60):
        got = []
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append([quantized_matmul(xs[(i + n) % 3], q, s, z, N) for _ in range(3)][-1])
        torch.cuda.synchronize()
        for n, o in enumerate(got):
            assert torch.equal(o, want[(i + n) % 3]), (i, n)

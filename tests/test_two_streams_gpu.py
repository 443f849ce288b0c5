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


@pytest.mark.parametrize("K,N,group", [
    (4096, 2048, 128),      # tcgen05
    (2048, 1024, 32),       # mma.sync with a ring
    (1024, 520, 64)])       # CUDA cores
@pytest.mark.parametrize("M", [1, 16, 33, 64, 65, 128, 129, 600])
def test_concurrent_products(M, K, N, group):
    from lightning_router.kernels.quantized_matmul import quantized_matmul
    from lightning_router.quantization.pack_weights import quantize_tensor
    g = torch.Generator().manual_seed(M)
    q, s, z = (v.to(DEV) for v in quantize_tensor(torch.randn(K, N, generator=g) * 0.02, group))
    xs = [torch.randn(M, K, generator=g).half().to(DEV) for _ in range(3)]
    want = []
    for x in xs:
        want.append(quantized_matmul(x, q, s, z, N, group))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(60):
        got = []
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append([quantized_matmul(xs[(i + n) % 3], q, s, z, N, group)
                            for _ in range(3)][-1])
        torch.cuda.synchronize()
        for n, o in enumerate(got):
            assert torch.equal(o, want[(i + n) % 3]), (i, n)


@pytest.mark.parametrize("R,requests,K,N,n,r", [
    (9600, 2, 256, 1544, 2, 8), (4099, 11, 512, 2056, 7, 32), (1111, 9, 2048, 1408, 6, 64),
    (200, 50, 520, 4104, 33, 16), (700, 700, 264, 264, 30, 128)])
def test_concurrent_adapters(R, requests, K, N, n, r):
    from lightning_router import _ext
    from lightning_router.kernels.adapters import AdapterBank, adapter_add, adapter_swiglu
    g = torch.Generator(device=DEV).manual_seed(R)

    def half(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=DEV) * std).half()
    bank = AdapterBank(half(n, r, K, std=K ** -0.5), half(n, N, r, std=0.2))
    sets = []
    for _ in range(3):
        ids = torch.randint(-1, n, (requests,), generator=g, device=DEV, dtype=torch.int32)
        sets.append((half(R, N), half(R, N), half(R, K),
                     ids.repeat_interleave(-(-R // requests))[:R].contiguous()))

    def both(base, up, x, ids):
        return (adapter_add(base, x, bank, ids),
                adapter_swiglu(base, up, x, bank, bank, ids))
    want = []
    for s in sets:
        want.append(both(*s))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(60):
        got = []
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(both(*sets[(i + k) % 3]))
        torch.cuda.synchronize()
        for k, o in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(o, want[(i + k) % 3])), (i, k)
    _ext.check_device_errors()


@pytest.mark.parametrize("T,d,E,k", [(64, 256, 8, 2), (777, 2048, 64, 6), (4000, 1024, 24, 4)])
def test_concurrent_training_steps(T, d, E, k):
    from lightning_router.kernels.routing_grad import (balanced_gating, combine_tokens,
                                                       dispatch_tokens, gate_projection)
    g = torch.Generator(device=DEV).manual_seed(T)
    w = torch.randn(E, d, generator=g, device=DEV) * 0.05
    sets = [torch.randn(T, d, generator=g, device=DEV).half() for _ in range(3)]

    def step(x):
        leaf, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
        logits = gate_projection(leaf, weight)
        plan = dispatch_tokens(leaf, logits, k, 0.9)
        out = combine_tokens(plan.permuted, plan.gate_weights, plan)
        loss = (out.float() ** 2).sum() / T + plan.aux_loss + balanced_gating(logits, k).aux_loss
        return torch.autograd.grad(loss, (leaf, weight))
    want = []
    for x in sets:
        want.append(step(x))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(30):
        got = []
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(step(sets[(i + n) % 3]))
        torch.cuda.synchronize()
        for n, o in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(o, want[(i + n) % 3])), (i, n)

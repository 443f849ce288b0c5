"""The adapters' second launch reads index, base rows and weights ahead of the first one's end:
every input may have been written by the kernel just before, in memory that an earlier call read."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("op", ["add", "swiglu"])
@pytest.mark.parametrize("R,requests,K,N,n,r", [
    (1, 1, 4096, 4096, 4, 8), (64, 64, 512, 4104, 64, 16), (256, 7, 256, 2056, 9, 64),
    (700, 700, 64, 264, 30, 16), (1111, 9, 512, 1408, 6, 64), (9600, 4, 64, 1544, 3, 32)])
def test_inputs_written_just_before(R, requests, K, N, n, r, op, in_place):
    from lightning_router import _ext
    from lightning_router.kernels.adapters import AdapterBank, adapter_add, adapter_swiglu
    g = torch.Generator(device=DEV).manual_seed(R + N)

    def half(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=DEV) * std).half()

    def case():
        ids = torch.randint(-1, n, (requests,), generator=g, device=DEV, dtype=torch.int32)
        return dict(x=half(R, K), base=half(R, N), up=half(R, N),
                    ids=ids.repeat_interleave(-(-R // requests))[:R].contiguous(),
                    a=half(n, r, K, std=K ** -0.5), b=half(n, N, r, std=0.2),
                    scale=torch.rand(n, generator=g, device=DEV) + 0.5)

    def call(t):
        bank = AdapterBank(t["a"], t["b"], t["scale"])
        out = t["base"] if in_place else None
        if op == "add":
            return adapter_add(t["base"], t["x"], bank, t["ids"], out=out)
        return adapter_swiglu(t["base"], t["up"], t["x"], bank, bank, t["ids"], out=out)

    cases = [case() for _ in range(3)]
    want = []
    for c in cases:
        want.append(call({k: v.clone() for k, v in c.items()}))
        torch.cuda.synchronize()
    now = {k: v.clone() for k, v in cases[0].items()}
    names = list(now)
    for i in range(60):
        c = cases[i % 3]
        got = []
        for last in (names[i % len(names)], names[(i + 3) % len(names)]):
            for k in names:                 # `last` is the youngest of the inputs
                if k != last:
                    now[k].copy_(c[k])
            now[last].copy_(c[last])
            got.append(call(now).clone())
        assert all(torch.equal(o, want[i % 3]) for o in got), i
    _ext.check_device_errors()

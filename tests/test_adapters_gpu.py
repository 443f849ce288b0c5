"""Low-rank adapters of many requests on the GPU against 64-bit products.

Tolerances are bounds by arithmetic: an fp16 store rounds by at most 2^-11 of the
value (2^-25 below the normal range), fp32 by 2^-24 (``U``); a tensor-core sum of n
steps is off by at most 4 n U times the sum of the terms' magnitudes (its adder may
truncate); v is split into two fp16 terms with 2^-22 of its row's largest left over.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _bank(g, n, r, K, N, scale=True):
    from lightning_router.kernels.adapters import AdapterBank
    return AdapterBank(_randn(g, n, r, K, std=K ** -0.5), _randn(g, n, N, r, std=0.2),
                       torch.rand(n, generator=g, device=DEV) * 2 - 0.5 if scale else None)


def delta64(x, bank, index):
    """(delta, its error bound) in double, adapter by adapter."""
    a, b, s = bank
    n, r, K = a.shape
    d = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(d)
    for i in range(n):
        t = torch.nonzero(index == i)[:, 0]
        if not t.numel():
            continue
        f = 1.0 if s is None else float(s[i])
        xa, aa, ba = x[t].double(), a[i].double(), b[i].double()
        v = xa @ aa.t()
        ev = (K // 16 + 80) * 4 * U * (xa.abs() @ aa.abs().t()) \
            + 4 * U * v.abs().amax(1, keepdim=True)
        d[t] = f * (v @ ba.t())
        tol[t] = abs(f) * (ev @ ba.abs().t() + (r // 4 + 8) * 4 * U * (v.abs() @ ba.abs().t()))
    return d, tol


def _check_add(out, base, x, bank, index):
    d, tol = delta64(x, bank, index)
    want = base.double() + d
    err = (out.double() - want).abs()
    tol = tol + 2 * U * want.abs() + want.abs() * 2.0 ** -11 + 2.0 ** -25
    assert bool((err <= tol).all()), (float((err - tol).max()), int((err > tol).sum()))
    none = (index < 0) | (index >= bank.a.shape[0])
    assert torch.equal(out[none], base[none])


def _rows(g, R, requests, n, without):
    """Contiguous requests of ragged lengths; some without an adapter."""
    if requests >= R:
        req = torch.arange(R, device=DEV)
    else:
        cuts = torch.randperm(R - 1, generator=g, device=DEV)[:requests - 1].sort().values + 1
        req = torch.searchsorted(cuts, torch.arange(R, device=DEV), right=True)
    ad = torch.randint(0, n, (int(req.max()) + 1,), generator=g, device=DEV)
    ad[torch.rand(ad.shape, generator=g, device=DEV) < without] = -1
    return ad[req].int()


SHAPES = [  # rows, requests, K, N, adapters, rank
    (1, 1, 8, 8, 1, 8), (1, 1, 4096, 4096, 4, 8), (2, 2, 40, 24, 3, 16), (7, 7, 64, 136, 9, 24),
    (8, 1, 512, 264, 2, 32), (9, 4, 1000, 1408, 5, 64), (17, 17, 256, 96, 20, 128),
    (64, 64, 1024, 2048, 64, 16), (65, 3, 72, 40, 2, 40), (200, 50, 520, 512, 33, 104),
    (256, 16, 2048, 256, 16, 16), (257, 5, 2048, 1000, 4, 16), (300, 300, 256, 256, 64, 32),
    (333, 9, 136, 8, 6, 64), (1111, 9, 2048, 1408, 6, 64), (1500, 2, 64, 2056, 2, 128),
    (4099, 11, 512, 512, 7, 32), (5000, 5000, 128, 64, 40, 16),
    # windows of 64 rows with streamed base rows: one, a few and many groups in a window
    (9600, 2, 64, 520, 2, 8), (4099, 11, 512, 1544, 7, 32), (3000, 40, 136, 1808, 33, 104),
    (2500, 9, 1000, 2056, 6, 64), (5000, 5000, 128, 1032, 40, 16), (19137, 700, 72, 232, 64, 24),
    # windows of 8 rows with many column groups to a warp; windows of 16 rows
    (256, 256, 64, 5000, 64, 16), (250, 1, 64, 9608, 2, 64), (129, 40, 72, 8200, 7, 32),
    (256, 30, 64, 4104, 9, 120), (700, 700, 64, 264, 30, 16), (500, 60, 64, 264, 9, 104)]


@pytest.mark.parametrize("R,requests,K,N,n,r", SHAPES)
@pytest.mark.parametrize("without", [0.0, 0.4])
def test_adapter_add(R, requests, K, N, n, r, without):
    from lightning_router import _ext
    from lightning_router.kernels.adapters import adapter_add
    g = _gen(R * 31 + K + r)
    x, base = _randn(g, R, K), _randn(g, R, N)
    bank = _bank(g, n, r, K, N, scale=without > 0)
    index = _rows(g, R, requests, n, without)
    out = adapter_add(base, x, bank, index)
    _check_add(out, base, x, bank, index)
    # the same in place, and again: the same bits
    again = base.clone()
    assert adapter_add(again, x, bank, index.long(), out=again).data_ptr() == again.data_ptr()
    assert torch.equal(again, out)
    _ext.check_device_errors()


def test_rows_in_any_order():
    """A row's result does not depend on its neighbours' adapters (up to the split of the sums
    over warps, which is within the bounds) nor on its place."""
    from lightning_router.kernels.adapters import adapter_add
    g = _gen(3)
    R, K, N, n, r = 900, 512, 264, 13, 16
    x, base, bank = _randn(g, R, K), _randn(g, R, N), _bank(g, n, r, K, N)
    index = _rows(g, R, 20, n, 0.2)
    perm = torch.randperm(R, generator=g, device=DEV)
    for order in (torch.arange(R, device=DEV), perm, torch.arange(R - 1, -1, -1, device=DEV)):
        out = adapter_add(base[order], x[order], bank, index[order])
        _check_add(out, base[order], x[order], bank, index[order])


@pytest.mark.parametrize("R", [24, 400, 19000])   # the last: streamed windows
def test_other_requests_infinities_stay_theirs(R):
    from lightning_router.kernels.adapters import AdapterBank, adapter_add
    g = _gen(4)
    K, N, n, r = 128, 64, 3, 16
    x, base, bank = _randn(g, R, K), _randn(g, R, N), _bank(g, n, r, K, N)
    index = (torch.arange(R, device=DEV) % 4 - 1).int()
    clean = adapter_add(base, x, bank, index)
    a, b = bank.a.clone(), bank.b.clone()
    a[1, 3, 5], b[1, 7, :] = float("nan"), float("inf")
    x2, base2 = x.clone(), base.clone()
    x2[index == -1] = float("nan")           # rows without an adapter do not read x
    base2[index == 1] = float("inf")
    out = adapter_add(base2, x2, AdapterBank(a, b, bank.scale), index)
    others = index != 1
    assert torch.equal(out[others], clean[others])
    assert not torch.isfinite(out[index == 1]).any()


@pytest.mark.parametrize("R", [40, 600])
def test_infinite_rows_are_infinite_where_the_products_are(R):
    """One infinity in a row of x: every product with it is infinite, of the sign of its factor
    (all of B positive, one element of A per rank not zero there)."""
    from lightning_router.kernels.adapters import AdapterBank, adapter_add
    g = _gen(14)
    K, N, r = 64, 512, 8
    x, base = _randn(g, R, K), _randn(g, R, N)
    a, b = _randn(g, 1, r, K), _randn(g, 1, N, r).abs() + 0.01
    a[0, :, 3] = 0.0
    a[0, 2, 3] = -1.0             # the infinity reaches one rank value only
    x[5, 3] = float("inf")
    index = torch.zeros(R, dtype=torch.int32, device=DEV)
    x[7] *= 600.0                 # a large finite row beside it
    out = adapter_add(base, x, AdapterBank(a, b), index)
    # 0 * inf is NaN in seven of the eight rank values, so the row is NaN as the formula's
    v = x.double() @ a[0].double().t()
    assert torch.isnan(v[5]).sum() == 7 and torch.isnan(out[5]).all()
    keep = torch.arange(R, device=DEV) != 5
    _check_add(out[keep], base[keep], x[keep], AdapterBank(a, b), index[keep])
    a[0, :, 3] = -1.0             # now all rank values are -inf
    out = adapter_add(base, x, AdapterBank(a, b), index)
    assert torch.equal(out[5], torch.full((N,), float("-inf"), device=DEV).half())


@pytest.mark.parametrize("magnitude", [1e-6, 1.0, 6e4])
def test_small_and_large_middle_values(magnitude):
    """v = x A^T far outside fp16 (up to 1e9, down to 1e-9) is not rounded to it."""
    from lightning_router.kernels.adapters import AdapterBank, adapter_add
    g = _gen(5)
    R, K, N, r = 40, 512, 64, 8
    x = _randn(g, R, K, std=min(magnitude, 1e4))
    a = _randn(g, 2, r, K, std=min(magnitude, 1e3))
    b = _randn(g, 2, N, r, std=1e-3 if magnitude > 1 else 1.0)
    scale = torch.tensor([1.0, 0.5], device=DEV)
    scale = scale * (1e-6 if magnitude > 1 else 1e9 if magnitude < 1 else 1.0)
    index = (torch.arange(R, device=DEV) % 2).int()
    base = _randn(g, R, N)
    bank = AdapterBank(a, b, scale)
    _check_add(adapter_add(base, x, bank, index), base, x, bank, index)


def test_bad_adapter_numbers_are_flagged_and_taken_as_none():
    from lightning_router import _ext
    from lightning_router.kernels.adapters import adapter_add
    g = _gen(6)
    x, base, bank = _randn(g, 5, 64), _randn(g, 5, 32), _bank(g, 3, 8, 64, 32)
    for index in (torch.tensor([0, 3, 2, -1, 1], device=DEV),
                  torch.tensor([0, -2, 2, -1, 1], device=DEV),
                  torch.tensor([0, 2**32, 2, -1, 1], device=DEV)):
        out = adapter_add(base, x, bank, index)
        with pytest.raises(RuntimeError, match="adapter"):
            _ext.check_device_errors()
        assert torch.equal(out[1], base[1]) and not torch.equal(out[0], base[0])
    _ext.check_device_errors()


@pytest.mark.parametrize("R,requests,K,N,n,r", [
    (1, 1, 64, 64, 1, 8), (5, 5, 72, 40, 3, 16), (128, 64, 1024, 1408, 64, 16),
    (100, 7, 256, 520, 4, 128), (257, 4, 512, 264, 8, 32), (1000, 20, 136, 96, 16, 48),
    # windows of 32 rows with streamed base rows
    (2001, 3, 256, 1288, 3, 16), (1500, 90, 136, 1800, 7, 24), (1100, 1100, 64, 2312, 40, 40),
    (9000, 12, 520, 264, 5, 128),
    # windows of 8 rows with many column groups to a warp; windows of 16 rows
    (200, 200, 64, 3208, 32, 16), (256, 100, 64, 4104, 7, 128), (255, 2, 64, 9608, 2, 32),
    (400, 130, 64, 264, 9, 16), (300, 6, 64, 264, 3, 128)])
def test_adapter_swiglu(R, requests, K, N, n, r):
    from lightning_router.kernels.adapters import adapter_swiglu
    g = _gen(R + K + N)
    x, gate, up = _randn(g, R, K), _randn(g, R, N, std=2.0), _randn(g, R, N)
    gb, ub = _bank(g, n, r, K, N), _bank(g, n, r, K, N, scale=False)
    index = _rows(g, R, requests, n, 0.25)
    out = adapter_swiglu(gate, up, x, gb, ub, index)
    dg, tg = delta64(x, gb, index)
    du, tu = delta64(x, ub, index)
    G, Uv = gate.double() + dg, up.double() + du
    tg, tu = tg + 2 * U * G.abs(), tu + 2 * U * Uv.abs()
    silu = G * torch.sigmoid(G)
    want = silu * Uv
    # |silu'| <= 1.1; the fast exponential and division are within 2^-20 + |G| 2^-22
    tol = 1.1 * tg * (Uv.abs() + tu) + silu.abs() * tu \
        + want.abs() * (2.0 ** -20 + G.abs() * 2.0 ** -22 + 2.0 ** -11) + 2.0 ** -25
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert torch.equal(adapter_swiglu(gate.clone(), up, x, gb, ub, index, out=gate), out)


def test_expert_row_numbers():
    from lightning_router import _ext
    from lightning_router.kernels.adapters import adapter_rows
    from lightning_router.kernels.expert_routing import topk_gating_dispatch
    g = _gen(7)
    T, E, k, n = 333, 16, 3, 5
    logits = _randn(g, T, E, dtype=torch.float32)
    logits[:, 4] = -1e30                     # an empty expert
    ad = torch.randint(-1, n, (T,), generator=g, device=DEV)
    plan = topk_gating_dispatch(_randn(g, T, 64), logits, k, 0.7)
    index = adapter_rows(ad, plan, n)
    offs, kept, src = plan.offsets.tolist(), plan.kept_counts.tolist(), plan.source_indices.tolist()
    a = ad.tolist()
    want = [-1] * (T * k)
    for e in range(E):
        for r in range(offs[e], offs[e] + kept[e]):
            if a[src[r]] >= 0:
                want[r] = a[src[r]] * E + e
    assert index.tolist() == want
    _ext.check_device_errors()
    adapter_rows(torch.full((T,), n, device=DEV), plan, n)
    with pytest.raises(RuntimeError, match="adapter"):
        _ext.check_device_errors()
    short = adapter_rows(ad[:100], plan, n)      # ids of another batch: flagged, not read past
    with pytest.raises(RuntimeError, match="source token"):
        _ext.check_device_errors()
    tokens = plan.source_indices
    assert torch.equal(short[tokens < 100], index[tokens < 100])
    assert bool((short[tokens >= 100] == -1).all())


def test_quantized_matmul_adapters():
    from lightning_router.kernels.adapters import adapter_add, quantized_matmul_adapters
    from lightning_router.kernels.quantized_matmul import quantized_matmul
    from lightning_router.quantization.pack_weights import quantize_tensor
    g = _gen(8)
    M, K, N = 96, 512, 256
    x, bank = _randn(g, M, K), _bank(g, 6, 16, K, N)
    q, s, z = quantize_tensor(_randn(g, K, N, std=0.05), 128)
    index = _rows(g, M, 10, 6, 0.3)
    out = quantized_matmul_adapters(x, q, s, z, N, bank, index)
    base = quantized_matmul(x, q, s, z, N)
    assert torch.equal(out, adapter_add(base, x, bank, index))
    _check_add(out, base, x, bank, index)


def test_strides_alignment_and_no_rows():
    from lightning_router.kernels.adapters import adapter_add
    g = _gen(9)
    R, K, N = 30, 64, 40
    bank = _bank(g, 3, 8, K, N)
    index = (torch.arange(R, device=DEV) % 3).int()
    wide = _randn(g, R, 2 * K)
    flat = _randn(g, 1 + R * N)
    x, base = wide[:, ::2], flat[1:].view(R, N)
    out = adapter_add(base, x, bank, index)
    assert torch.equal(out, adapter_add(base.clone(), x.contiguous(), bank, index))
    rows = torch.empty(2 * R, device=DEV, dtype=torch.int32)
    rows[::2] = index
    assert torch.equal(adapter_add(base, x, bank, rows[::2]), out)
    assert adapter_add(base[:0], x[:0], bank, index[:0]).shape == (0, N)
    from lightning_router.kernels.adapters import adapter_swiglu
    assert adapter_swiglu(base[:0], base[:0], x[:0], bank, bank, index[:0]).shape == (0, N)


def test_streams_and_graphs():
    from lightning_router.kernels.adapters import adapter_add
    g = _gen(10)
    R, K, N = 48, 256, 512
    x, base, bank = _randn(g, R, K), _randn(g, R, N), _bank(g, 48, 16, K, N)
    index = torch.arange(R, device=DEV).int()
    ref = adapter_add(base, x, bank, index)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [adapter_add(base, x, bank, index) for _ in range(3)]
    here = [adapter_add(base, x, bank, index) for _ in range(3)]   # at the same time
    torch.cuda.current_stream().wait_stream(side)
    for o in outs + here:
        assert torch.equal(o, ref)
    graphs, got = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got.append(adapter_add(base, x, bank, index))
        graphs.append(gr)
    index.copy_(torch.randperm(R, generator=g, device=DEV))
    x.copy_(_randn(g, R, K))
    for gr in graphs:
        gr.replay()
    ref = adapter_add(base, x, bank, index)
    assert torch.equal(got[0], ref) and torch.equal(got[1], ref)


def test_pack_adapters_of_different_ranks():
    from lightning_router.kernels.adapters import adapter_add, pack_adapters
    g = _gen(11)
    K, N = 64, 48
    pairs = [(_randn(g, r, K, std=0.1), _randn(g, N, r)) for r in (4, 16, 11)]
    bank = pack_adapters(pairs, [1.0, 2.0, 0.5])
    assert bank.a.shape == (3, 16, K) and bank.b.shape == (3, N, 16)
    x, base = _randn(g, 3, K), _randn(g, 3, N)
    index = torch.tensor([2, 0, 1], device=DEV)
    out = adapter_add(base, x, bank, index)
    _check_add(out, base, x, bank, index)
    A, B = pairs[2]
    want = base[0].double() + 0.5 * (x[0].double() @ A.double().t()) @ B.double().t()
    assert float((out[0].double() - want).abs().max()) <= 2.0 ** -9 * float(want.abs().max())


def test_refusals():
    from lightning_router.kernels.adapters import AdapterBank, adapter_add, adapter_swiglu
    g = _gen(12)
    x, base, bank = _randn(g, 4, 64), _randn(g, 4, 32), _bank(g, 2, 8, 64, 32)
    index = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="index"):
        adapter_add(base, x, bank, index[:3])
    with pytest.raises(ValueError, match="integers"):
        adapter_add(base, x, bank, index.float())
    with pytest.raises(RuntimeError, match="base"):
        adapter_add(base[:, :24], x, bank, index)
    with pytest.raises(RuntimeError, match="columns"):
        adapter_add(base, x[:, :56], bank, index)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        adapter_add(base, x, AdapterBank(bank.a[:, :4].contiguous(), bank.b[:, :, :4].contiguous()),
                    index)
    with pytest.raises(RuntimeError, match="contiguous"):
        adapter_add(base, x, AdapterBank(bank.a.transpose(1, 2).contiguous().transpose(1, 2),
                                         bank.b), index)
    with pytest.raises(RuntimeError, match="at most 128"):
        adapter_add(base, x, _bank(g, 1, 136, 64, 32), index)
    buf = torch.zeros(5, 32, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        adapter_add(buf[:4], x, bank, index, out=buf[1:])
    with pytest.raises(RuntimeError, match="no backward"):
        adapter_add(base, x.clone().requires_grad_(), bank, index)
    with pytest.raises(RuntimeError, match="differ in size"):
        adapter_swiglu(base, base, x, bank, _bank(g, 2, 16, 64, 32), index)

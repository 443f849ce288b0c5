"""The router's training path on the GPU against 64-bit formulas.

Tolerances are bounds by arithmetic.  fp32 steps round by at most 2^-24 of their
result (``U``); an accumulation of n terms is off by at most n U times the sum of
their magnitudes, a tensor-core one by at most four times that (its adder may
truncate); an fp16 store by 2^-11 of the value or 2^-25 below the normal range.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
LBW = 0.01


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _close(got, want, tol, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want.double()).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(err[bad].max()),
                                 float((torch.as_tensor(tol, device=err.device)
                                        .expand_as(err))[bad].min()))


def _half_tol(want):
    return want.abs() * 2.0 ** -11 + 2.0 ** -25


# ---------------------------------------------------------------------------
# balanced gating
# ---------------------------------------------------------------------------
def gating64(logits, k, mask, lbw=LBW):
    """ids, p, weights, q, counts, aux of the definition in double."""
    T, E = logits.shape
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    p = torch.softmax(logits.double(), 1)
    ps = p.gather(1, ids)
    q = ps.sum(1, keepdim=True) + 1e-9
    w = ps / q
    live = torch.ones(T, dtype=torch.bool, device=logits.device) if mask is None else mask
    n = int(live.sum())
    counts = torch.bincount(ids[live].reshape(-1), minlength=E)
    f = counts.double() / max(n * k, 1)
    aux = lbw * E * (f * p[live].sum(0) / max(n, 1)).sum()
    return ids, p, torch.where(live[:, None], w, 0.0), q, counts, aux, f, live, n


def gating_grad64(logits, k, mask, dw, da, lbw=LBW):
    ids, p, w, q, counts, _, f, live, n = gating64(logits, k, mask, lbw)
    T, E = logits.shape
    w = p.gather(1, ids) / q
    dw = dw.double().view(T, k)
    c = (dw * w).sum(1, keepdim=True)
    dp = torch.zeros_like(p).scatter_add(1, ids, (dw - c) / q)
    bal = float(da) * lbw * E * f / max(n, 1)
    dp = dp + bal
    dl = p * (dp - (p * dp).sum(1, keepdim=True))
    scale = p * ((dw.abs().amax(1, keepdim=True) + c.abs()) / q + bal.abs().max()) * 2
    return torch.where(live[:, None], dl, 0.0), scale


def _spread(logits):
    return (logits.amax(1, keepdim=True) - logits.amin(1, keepdim=True)).double()


GATING = [(5, 1, 1), (1, 2, 1), (1, 64, 8), (7, 3, 3), (31, 5, 2), (64, 8, 2), (300, 16, 4), (333, 17, 5),
          (512, 32, 8), (513, 33, 1), (1000, 64, 6), (4097, 61, 7), (70001, 8, 2), (40000, 64, 6)]


@pytest.mark.parametrize("T,E,k", GATING)
@pytest.mark.parametrize("padded", [0.0, 0.4])
def test_balanced_gating(T, E, k, padded):
    from lightning_router.kernels.routing_grad import balanced_gating
    g = _gen(T * 131 + E)
    logits = _randn(g, T, E, std=1.5)
    mask = (torch.rand(T, generator=g, device=DEV) >= padded) if padded else None
    leaf = logits.clone().requires_grad_()
    out = balanced_gating(leaf, k, LBW, mask)
    ids, p, w, q, counts, aux, *_ = gating64(logits, k, mask)
    assert torch.equal(out.expert_ids.view(T, k).long(), ids)
    assert torch.equal(out.expert_counts.long(), counts)
    eps = (_spread(logits) + E + 32) * 2 * U   # exp of a rounded difference, sums of E terms
    _close(out.gate_weights.view(T, k), w, w * eps + 1e-30, "weights")
    assert abs(float(out.aux_loss.detach()) - float(aux)) <= float(eps.max()) * abs(float(aux)) + 1e-30
    dw, da = _randn(g, T * k), torch.tensor(float(T) * 3, device=DEV)
    (dl,) = torch.autograd.grad((out.gate_weights, out.aux_loss), leaf, (dw, da))
    want, scale = gating_grad64(logits, k, mask, dw, da)
    _close(dl, want, scale * eps * 2 + 1e-30, "d_logits")


def test_balanced_gating_one_output_only():
    from lightning_router.kernels.routing_grad import balanced_gating
    g = _gen(5)
    logits = _randn(g, 100, 12)
    zero_w, zero_a = torch.zeros(300, device=DEV), torch.zeros((), device=DEV)
    for pick in ("weights", "aux"):
        leaf = logits.clone().requires_grad_()
        out = balanced_gating(leaf, 3)
        if pick == "weights":
            dw, da = _randn(g, 300), zero_a
            out.gate_weights.backward(dw)
        else:
            dw, da = zero_w, torch.ones((), device=DEV)
            out.aux_loss.backward()
        want, scale = gating_grad64(logits, 3, None, dw, da)
        _close(leaf.grad, want, scale * (_spread(logits) + 44) * 4 * U, pick)


def test_balanced_gating_ties_infinities_and_nan_in_padding():
    from lightning_router.kernels.routing_grad import balanced_gating
    logits = torch.zeros(6, 8, device=DEV)
    logits[1, 3:] = 1.0                       # ties among the largest
    logits[2, 1::2] = float("-inf")           # experts switched off
    logits[3] = torch.tensor([0.0, -0.0] * 4)  # equal zeros of both signs
    logits[4] = float("nan")
    logits[5] = float("-inf")
    mask = torch.tensor([True, True, True, True, False, False], device=DEV)
    leaf = logits.clone().requires_grad_()
    out = balanced_gating(leaf, 2, LBW, mask)
    assert out.expert_ids.view(6, 2).tolist()[:4] == [[0, 1], [3, 4], [0, 2], [0, 1]]
    assert all(0 <= a < 8 and 0 <= b < 8 and a != b for a, b in out.expert_ids.view(6, 2).tolist())
    assert out.gate_weights[8:].tolist() == [0.0] * 4
    assert out.expert_counts.tolist() == [3, 2, 1, 1, 1, 0, 0, 0]
    assert torch.isfinite(out.aux_loss)
    out.aux_loss.backward()
    assert torch.isfinite(leaf.grad).all() and not leaf.grad[4:].any()
    # nothing live: no loss, no gradient
    leaf = logits.clone().requires_grad_()
    out = balanced_gating(leaf, 2, LBW, torch.zeros(6, dtype=torch.bool, device=DEV))
    assert float(out.aux_loss.detach()) == 0.0 and not out.expert_counts.any()
    out.aux_loss.backward()
    assert not leaf.grad.any()


def test_balanced_gating_no_tokens_and_strides():
    from lightning_router.kernels.routing_grad import balanced_gating
    leaf = torch.zeros(0, 8, device=DEV, requires_grad=True)
    out = balanced_gating(leaf, 2)
    assert out.expert_ids.numel() == 0 and float(out.aux_loss.detach()) == 0 and out.expert_counts.sum() == 0
    out.aux_loss.backward()
    assert leaf.grad.shape == (0, 8)
    wide = _randn(_gen(1), 50, 40)
    leaf = wide.clone().requires_grad_()
    out = balanced_gating(leaf[:, 3:36:2], 2)     # 17 strided columns
    ref = balanced_gating(wide[:, 3:36:2].contiguous(), 2)
    assert torch.equal(out.gate_weights, ref.gate_weights)
    out.gate_weights.sum().backward()             # an expanded gradient
    assert torch.isfinite(leaf.grad).all() and not leaf.grad[:, 0].any()


def test_balanced_gating_matches_inference_gating():
    from lightning_router.kernels.expert_routing import topk_gating_dispatch
    from lightning_router.kernels.routing_grad import balanced_gating
    logits = _randn(_gen(2), 2048, 64)
    a, b = balanced_gating(logits, 6), topk_gating_dispatch(None, logits, 6)
    assert torch.equal(a.expert_ids, b.expert_ids)
    _close(a.gate_weights, b.gate_weights, 200 * U * b.gate_weights.double())
    assert torch.equal(a.expert_counts, b.offsets.diff())
    assert abs(float(a.aux_loss) - float(b.aux_loss)) <= 200 * U * float(b.aux_loss)


def test_balanced_gating_gradient_against_differences():
    """The gradient along a direction against central differences of the 64-bit loss: the step
    is small enough for no selection to change (checked)."""
    from lightning_router.kernels.routing_grad import balanced_gating
    g = _gen(9)
    T, E, k = 40, 10, 3
    logits, v = _randn(g, T, E), _randn(g, T, E)
    dw = _randn(g, T * k)
    leaf = logits.clone().requires_grad_()
    out = balanced_gating(leaf, k, 1.0)
    loss = (out.gate_weights * dw).sum() + 5.0 * out.aux_loss
    loss.backward()
    got = float((leaf.grad.double() * v.double()).sum())
    ids = gating64(logits, k, None)[0]

    def value(x):
        p = torch.softmax(x, 1)
        ps = p.gather(1, ids)
        w = ps / (ps.sum(1, keepdim=True) + 1e-9)
        f = torch.bincount(ids.reshape(-1), minlength=E).double() / (T * k)
        return float((w.reshape(-1) * dw.double()).sum() + 5.0 * E * (f * p.mean(0)).sum())

    h = 1e-5
    x, d = logits.double(), v.double()
    for s in (h, -h):
        assert torch.equal(torch.sort(x + s * d, dim=1, descending=True, stable=True).indices[:, :k], ids)
    want = (value(x + h * d) - value(x - h * d)) / (2 * h)
    # differences: h^2 times third derivatives (order of the value, 1e2) and 2^-53 * value / h
    scale = float((leaf.grad.double() * v.double()).abs().sum())
    assert abs(got - want) <= 1e-7 + scale * 200 * U


@pytest.mark.parametrize("T,E,k", [(20000, 2, 1), (50000, 8, 1), (30000, 64, 1), (4000, 5, 2)])
def test_balanced_gating_gradient_of_a_balanced_router(T, E, k):
    """Nearly equal counts, weights of (nearly) 1: the gradient is a difference of nearly equal
    terms, which is taken before it is rounded."""
    from lightning_router.kernels.routing_grad import balanced_gating
    g = _gen(T + E)
    logits = _randn(g, T, E)
    dw, da = _randn(g, T * k, std=1.0 / T), torch.ones((), device=DEV)
    if k == 2:
        logits[:, 0] += 18.0        # one expert has all of the weight
    leaf = logits.clone().requires_grad_()
    out = balanced_gating(leaf, k)
    (dl,) = torch.autograd.grad((out.gate_weights, out.aux_loss), leaf, (dw, da))
    # differences of dw and counts are exact or rounded once: the error is that of p alone,
    # in relation to the gradient itself: the exact form from 64-bit differences
    ids, p, w, q, counts, _, f, _, n = gating64(logits, k, None)
    d = dw.double().view(T, k)
    d0 = d[:, :1]
    bal = LBW * E * (f - 1.0 / E) / n
    rest = (((d - d0) * (p.gather(1, ids) / q)).sum(1, keepdim=True) - d0 * 1e-9 / q) / q
    dp = (bal[None, :] - bal[ids[:, :1]]) + rest.expand(T, E).scatter(1, ids, (d - d0) / q)
    want = p * (dp - (p * dp).sum(1, keepdim=True))
    eps = float(_spread(logits).max()) + E + 32
    assert float((dl.double() - want).norm() / want.norm()) <= eps * 4 * U


# ---------------------------------------------------------------------------
# gate projection
# ---------------------------------------------------------------------------
GATE = [(1, 16, 1), (3, 48, 5), (17, 64, 8), (64, 80, 9), (256, 496, 64), (100, 64, 70), (255, 4096, 7), (100, 1024, 4), (257, 208, 16),
        (1000, 512, 33), (4000, 1264, 24), (3001, 2000, 100), (2049, 256, 64), (5000, 2048, 8), (300, 64, 130), (6000, 1040, 64)]


@pytest.mark.parametrize("T,d,E", GATE)
@pytest.mark.parametrize("master", [True, False])
def test_gate_projection(T, d, E, master):
    from lightning_router.kernels.expert_routing import gate_logits
    from lightning_router.kernels.routing_grad import gate_projection
    g = _gen(T + d + E)
    h = _randn(g, T, d, dtype=torch.float16).requires_grad_()
    w = _randn(g, E, d, std=0.05, dtype=torch.float32 if master else torch.float16).requires_grad_()
    b = _randn(g, E).requires_grad_()
    dl = _randn(g, T, E, std=1e-5 if master else 1.0)   # small ones keep their bits too
    out = gate_projection(h, w, b)
    assert torch.equal(out.detach(), gate_logits(h.detach(), w.detach(), b.detach()))
    dh, dw, db = torch.autograd.grad(out, (h, w, b), dl)
    assert dh.dtype == h.dtype and dw.dtype == w.dtype and db.dtype == torch.float32
    h64, w64, d64 = h.detach().double(), w.detach().half().double(), dl.double()
    want = d64 @ w64
    _close(dh, want, _half_tol(want) + (E // 4 + 8) * 4 * U * (d64.abs() @ w64.abs()), "dh")
    want = d64.t() @ h64
    # split 2^-22, a chain of 64 tensor-core sums, 8 warps, the token ranges
    tol = (64 + 8 + T // 128 + 8) * 4 * U * (d64.abs().t() @ h64.abs())
    _close(dw, want, tol if master else tol + _half_tol(want), "dw")
    _close(db, d64.sum(0), (T // 4 + 64) * U * d64.abs().sum(0) + 1e-30, "db")


def test_gate_projection_parts_and_empty():
    from lightning_router.kernels.routing_grad import gate_projection
    g = _gen(3)
    h, w = _randn(g, 40, 64, dtype=torch.float16), _randn(g, 6, 64)
    full = [h.clone().requires_grad_(), w.clone().requires_grad_()]
    dl = _randn(g, 40, 6)
    dh, dw = torch.autograd.grad(gate_projection(*full), full, dl)
    hr = h.clone().requires_grad_()
    (a,) = torch.autograd.grad(gate_projection(hr, w), hr, dl)
    wr = w.clone().requires_grad_()
    (b,) = torch.autograd.grad(gate_projection(h, wr), wr, dl)
    br = torch.zeros(6, device=DEV, requires_grad=True)
    (c,) = torch.autograd.grad(gate_projection(h, w, br), br, dl)
    assert torch.equal(a, dh) and torch.equal(b, dw)
    _close(c, dl.double().sum(0), 64 * U * dl.double().abs().sum(0))
    e = torch.zeros(0, 64, dtype=torch.float16, device=DEV, requires_grad=True)
    wr = w.clone().requires_grad_()
    out = gate_projection(e, wr)
    assert out.shape == (0, 6)
    out.sum().backward()
    assert not wr.grad.any() and e.grad.shape == (0, 64)


def test_gate_projection_rounds_the_master_weight_as_torch_does():
    from lightning_router.kernels.routing_grad import gate_projection
    g = _gen(6)
    h = torch.eye(64, device=DEV).half()            # logits are the weight's columns
    w = _randn(g, 9, 64) * torch.logspace(-9, 6, 64, device=DEV)   # subnormal to infinite in fp16
    w[0, :4] = torch.tensor([1 + 2.0**-11, 1 + 3 * 2.0**-11, 65519.0, 65520.0], device=DEV)
    w2 = torch.where(torch.isfinite(w.half()), w, 0.0)
    assert torch.equal(gate_projection(h, w2), w2.half().float().t())
    assert torch.equal(gate_projection(h, w2[:, ::1].half()), gate_projection(h, w2))


def test_gate_projection_unaligned_and_strided_rows():
    from lightning_router.kernels.routing_grad import gate_projection
    g = _gen(4)
    flat = _randn(g, 1 + 30 * 64, dtype=torch.float16)
    w = _randn(g, 6, 64).requires_grad_()
    dl = _randn(g, 30, 6)
    odd = flat[1:].view(30, 64)                   # 2-byte aligned rows
    (a,) = torch.autograd.grad(gate_projection(odd, w), w, dl)
    (b,) = torch.autograd.grad(gate_projection(odd.clone(), w), w, dl)
    assert torch.equal(a, b)
    wide = _randn(g, 30, 128, dtype=torch.float16).requires_grad_()
    out = gate_projection(wide[:, ::2], w)
    (dwide,) = torch.autograd.grad(out, wide, dl)
    assert not dwide[:, 1::2].any() and dwide[:, ::2].any()


# ---------------------------------------------------------------------------
# dispatch and combine
# ---------------------------------------------------------------------------
ROUTE = [(1, 8, 2, 1, 1.25), (1, 64, 8, 8, 1.0), (5, 24, 3, 2, 0.5), (64, 4096, 8, 2, 1.25),
         (257, 520, 4, 2, 1.0), (333, 1032, 64, 6, 0.5), (2500, 256, 8, 2, 0.7),
         (3000, 72, 16, 1, 10.0), (700, 2048, 64, 8, 0.1)]


@pytest.mark.parametrize("T,d,E,k,cf", ROUTE)
def test_dispatch_and_combine(T, d, E, k, cf):
    from lightning_router.kernels.expert_routing import combine, topk_gating_dispatch
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    g = _gen(T + d * 7 + E)
    S = T * k
    x = _randn(g, T, d, dtype=torch.float16).requires_grad_()
    logits = _randn(g, T, E).requires_grad_()
    y = _randn(g, S, d, dtype=torch.float16).requires_grad_()
    dout, dperm = _randn(g, T, d, dtype=torch.float16), _randn(g, S, d, dtype=torch.float16)
    da = torch.tensor(100.0, device=DEV)
    plan = dispatch_tokens(x, logits, k, cf, LBW)
    out = combine_tokens(y, plan.gate_weights, plan)
    ref = topk_gating_dispatch(x.detach(), logits.detach(), k, cf, LBW, fill_dropped=True)
    for name in ref._fields:
        a, b = getattr(plan, name), getattr(ref, name)
        assert a == b if name == "capacity" else torch.equal(a.detach(), b), name
    assert torch.equal(out.detach(), combine(y.detach(), ref.gate_weights, ref.slot_pos, T, k))
    dx, dl, dy = torch.autograd.grad((out, plan.permuted, plan.aux_loss), (x, logits, y),
                                     (dout, dperm, da))
    pos = ref.slot_pos.long()
    kept = (pos >= 0)
    w64, y64, do64 = ref.gate_weights.double(), y.detach().double(), dout.double()
    tok = torch.arange(S, device=DEV) // k
    rows = torch.where(kept[:, None], dperm.double()[pos.clamp(min=0)], 0.0).view(T, k, d)
    want = rows.sum(1)
    _close(dx, want, _half_tol(want) + k * 2 * U * rows.abs().sum(1), "dx")
    want = torch.zeros(S, d, dtype=torch.float64, device=DEV)
    want[pos[kept]] = (w64[:, None] * do64[tok])[kept]
    _close(dy, want, _half_tol(want) + 2 * U * want.abs(), "dy")
    prod = do64[tok] * y64[pos.clamp(min=0)]
    dw = torch.where(kept, prod.sum(1), 0.0)
    dw_tol = torch.where(kept, prod.abs().sum(1), 0.0) * d * U
    want, scale = gating_grad64(logits.detach(), k, None, dw, da)
    _, p, w, q, *_ = gating64(logits.detach(), k, None)
    tol = scale * (_spread(logits.detach()) + E + 32) * 4 * U
    # the weights' own gradients are off by dw_tol: through the formula's absolute values
    tol = tol + 4 * p * (dw_tol.view(T, k).amax(1, keepdim=True) / q)
    _close(dl, want, tol + 1e-30, "dl")


def test_combine_weights_gradient_alone_and_detached_rows():
    """Frozen experts: the rows need no gradient, the weights do."""
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    g = _gen(8)
    T, d, E, k = 90, 128, 4, 2
    x = _randn(g, T, d, dtype=torch.float16)
    logits = _randn(g, T, E).requires_grad_()
    plan = dispatch_tokens(x, logits, k, 0.6)
    assert plan.permuted.shape == (T * k, d)
    y = _randn(g, T * k, d, dtype=torch.float16)
    w = plan.gate_weights.detach().requires_grad_()
    out = combine_tokens(y, w, plan)
    dout = _randn(g, T, d, dtype=torch.float16)
    (dw,) = torch.autograd.grad(out, w, dout)
    pos = plan.slot_pos.long()
    prod = dout.double()[torch.arange(T * k, device=DEV) // k] * y.double()[pos.clamp(min=0)]
    prod = torch.where((pos >= 0)[:, None], prod, 0.0)
    _close(dw, prod.sum(1), prod.abs().sum(1) * d * U)
    assert bool((pos < 0).any()) and not dw[pos < 0].any()


def test_row_gradients_against_differences():
    """combine is linear in rows and weights, dispatch in the rows: a difference is exact up
    to rounding.  <dy, v> against <dout, combine(v)> and <dx, v> against <dperm, dispatch(v)>."""
    from lightning_router.kernels.routing_grad import combine_tokens, dispatch_tokens
    g = _gen(11)
    T, d, E, k = 200, 64, 8, 2
    logits = _randn(g, T, E)
    x = _randn(g, T, d, dtype=torch.float16).requires_grad_()
    y = _randn(g, T * k, d, dtype=torch.float16).requires_grad_()
    plan = dispatch_tokens(x, logits, k, 0.8)
    w = plan.gate_weights.detach()
    dout, dperm = _randn(g, T, d, dtype=torch.float16), _randn(g, T * k, d, dtype=torch.float16)
    dx, dy = torch.autograd.grad((combine_tokens(y, w, plan), plan.permuted), (x, y), (dout, dperm))
    vy, vx = _randn(g, T * k, d, dtype=torch.float16), _randn(g, T, d, dtype=torch.float16)
    with torch.no_grad():
        cy = combine_tokens(vy, w, plan).double()
        px = dispatch_tokens(vx, logits, k, 0.8).permuted.double()
    for a, b, c, e in ((dy, vy, dout, cy), (dx, vx, dperm, px)):
        left, right = (a.double() * b.double()), (c.double() * e)
        tol = 2.0 ** -10 * (left.abs().sum() + right.abs().sum()) + 1e-3
        assert abs(float(left.sum() - right.sum())) <= float(tol)


# ---------------------------------------------------------------------------
# how they are called
# ---------------------------------------------------------------------------
def _step(x, logits, w, h, k=2):
    from lightning_router.kernels.routing_grad import (combine_tokens, dispatch_tokens,
                                                       gate_projection)
    lg = gate_projection(h, w) + logits
    plan = dispatch_tokens(x, lg, k, 1.0)
    out = combine_tokens(plan.permuted * 2, plan.gate_weights, plan)
    return (out.float() ** 2).mean() + plan.aux_loss


def test_gradients_are_deterministic_and_on_another_stream():
    g = _gen(21)
    T, d, E = 600, 256, 16
    x, h = (_randn(g, T, d, dtype=torch.float16).requires_grad_() for _ in range(2))
    logits, w = _randn(g, T, E), _randn(g, E, d, std=0.05).requires_grad_()
    ref = torch.autograd.grad(_step(x, logits, w, h), (x, w, h))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(_step(x, logits, w, h), (x, w, h))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(ref, got):
        assert torch.equal(a, b)


def test_forward_and_backward_in_a_graph():
    g = _gen(22)
    T, d, E = 300, 128, 8
    x, h = (_randn(g, T, d, dtype=torch.float16).requires_grad_() for _ in range(2))
    logits, w = _randn(g, T, E), _randn(g, E, d, std=0.05).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(_step(x, logits, w, h), (x, w, h))
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):      # two graphs, each with its own workspaces
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(torch.autograd.grad(_step(x, logits, w, h), (x, w, h)))
        graphs.append(gr)
    with torch.no_grad():
        logits.copy_(_randn(g, T, E))
        x.copy_(_randn(g, T, d, dtype=torch.float16))
    for gr in graphs:
        gr.replay()
    ref = torch.autograd.grad(_step(x, logits, w, h), (x, w, h))
    for got in outs:
        for a, b in zip(ref, got):
            assert torch.equal(a, b)


def test_no_graph_is_recorded_where_none_is_wanted():
    from lightning_router.kernels.routing_grad import balanced_gating, gate_projection
    leaf = torch.randn(8, 4, device=DEV, requires_grad=True)
    with torch.no_grad():
        assert not balanced_gating(leaf, 2).aux_loss.requires_grad
    with torch.inference_mode():
        assert not balanced_gating(leaf, 2).gate_weights.requires_grad
        assert gate_projection(torch.randn(2, 16, device=DEV), torch.randn(3, 16, device=DEV)).shape \
            == (2, 3)


def test_refusals():
    from lightning_router.kernels.routing_grad import (balanced_gating, combine_tokens,
                                                       dispatch_tokens, gate_projection)
    lg = torch.randn(8, 4, device=DEV)
    with pytest.raises(RuntimeError, match="E <= 64"):
        balanced_gating(torch.randn(8, 65, device=DEV), 2)
    for k in (0, 5):
        with pytest.raises(RuntimeError, match="k"):
            balanced_gating(lg, k)
    with pytest.raises(RuntimeError, match="token_mask"):
        balanced_gating(lg, 2, token_mask=torch.ones(7, dtype=torch.bool, device=DEV))
    with pytest.raises(RuntimeError, match="token_mask"):
        balanced_gating(lg, 2, token_mask=torch.ones(8, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA"):
        balanced_gating(lg, 2, token_mask=torch.ones(8, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="invalid argument"):
        gate_projection(torch.randn(4, 24, device=DEV), torch.randn(3, 24, device=DEV))
    with pytest.raises(RuntimeError, match="expected"):
        gate_projection(torch.randn(4, 32, device=DEV), torch.randn(3, 16, device=DEV))
    x = torch.randn(8, 16, device=DEV).half()
    plan = dispatch_tokens(x, lg, 2)
    with pytest.raises(RuntimeError, match="one fp16 row per slot"):
        combine_tokens(plan.permuted[:-1], plan.gate_weights, plan)
    with pytest.raises(RuntimeError, match="gate_weights"):
        combine_tokens(plan.permuted, plan.gate_weights.half(), plan)
    leaf = lg.clone().requires_grad_()
    out = balanced_gating(leaf, 2)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out.aux_loss, leaf, create_graph=True)

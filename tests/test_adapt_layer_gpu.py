"""The layer with adapters and with gradients: the operators run together as a user runs them.

``MoELayer.forward(h, adapter_ids=...)`` against a 64-bit layer with the adapters added to the
dequantized weights' products; the trainable layer's router gradient over frozen INT4 experts
and all gradients over plain experts against 64-bit autograd of the same layer.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _workload(name="decode", **kw):
    from lightning_router.workloads import WORKLOADS
    return dataclasses.replace(WORKLOADS[name], **kw)


def _adapters(layer, n, rank, seed, std=0.05):
    from lightning_router.models.adapters import ExpertAdapters
    ad = ExpertAdapters(n, layer.num_experts, layer.hidden_size, layer.intermediate_size, rank,
                        gated=layer.experts.activation == "swiglu").to(DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for m in ad.mats:
        a, b = getattr(ad, f"{m}_a"), getattr(ad, f"{m}_b")
        a.copy_(torch.randn(a.shape, generator=g, device=DEV) * a.shape[-1] ** -0.5)
        b.copy_(torch.randn(b.shape, generator=g, device=DEV) * std)
        s = getattr(ad, f"{m}_scale")
        s.copy_(torch.rand(s.shape, generator=g, device=DEV) + 0.5)
    return ad


def _layer64(layer, t, w, plan, x, ids):
    """The layer in double on the kernel's routing plan, adapters by (adapter, expert)."""
    from lightning_router.quantization.pack_weights import dequantize_tensor
    ad = layer.adapters
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    offs, kept = plan.offsets.tolist(), plan.kept_counts.tolist()

    def product(rows, W, mat, e, a):
        o = rows @ W
        for i in range(ad.num_adapters):
            r = torch.nonzero(a == i)[:, 0]
            A = getattr(ad, f"{mat}_a")[i, e].double()
            B = getattr(ad, f"{mat}_b")[i, e].double()
            o[r] += float(getattr(ad, f"{mat}_scale")[i, e]) * (rows[r] @ A.t()) @ B.t()
        return o

    for e, ex in enumerate(t.experts):
        rows = slice(offs[e], offs[e] + kept[e])
        toks = plan.source_indices[rows].long()
        W = {m: dequantize_tensor(q, s, z, w.group_size, s.shape[1]).double()
             for m, (q, s, z) in ex.items()}
        xe, a = x[toks].double(), ids[toks]
        up = product(xe, W["up"], "up", e, a)
        if "gate" in W:
            h = torch.nn.functional.silu(product(xe, W["gate"], "gate", e, a)) * up
        else:
            h = torch.nn.functional.silu(up)
        out.index_add_(0, toks, product(h, W["down"], "down", e, a)
                       * plan.routing_weights[rows, None].double())
    return out


@pytest.mark.parametrize("name,overrides,n,rank", [
    ("decode", dict(d_model=512, d_ff=1024), 4, 16),
    ("decode", dict(d_model=512, d_ff=1024, tokens=1), 2, 8),
    ("fine", dict(tokens=300, d_model=256, d_ff=256), 3, 8),
    ("prefill", dict(tokens=1500, d_model=256, d_ff=512, capacity_factor=0.7), 5, 32),
    ("pr1", dict(tokens=200, d_model=256, d_ff=384), 3, 16),
])
def test_layer_with_adapters(name, overrides, n, rank):
    from lightning_router import _ext
    from lightning_router.workloads import build_layer
    w = _workload(name, **overrides)
    layer, t = build_layer(w, device=DEV)
    plain, aux0 = layer(t.x)
    layer.adapters = _adapters(layer, n, rank, 3)
    g = torch.Generator(device=DEV).manual_seed(5)
    ids = torch.randint(-1, n, (max(1, w.tokens // 7),), generator=g, device=DEV)
    ids = ids.repeat_interleave(-(-w.tokens // ids.numel()))[:w.tokens]   # runs of a request
    out, aux = layer(t.x, adapter_ids=ids)
    assert torch.equal(aux, aux0)
    _, plan = layer.route(t.x)
    ref = _layer64(layer, t, w, plan, t.x, ids)
    # the INT4 layer's own bound (1e-3) and four more fp16 roundings of at most 2^-11
    assert float((out.double() - ref).norm() / ref.norm()) <= 1e-3 + 2 * 2.0 ** -11
    again, _ = layer(t.x, adapter_ids=ids)
    assert torch.equal(out, again)
    assert torch.equal(layer(t.x)[0], plain)        # without ids: as before
    _ext.check_device_errors()


def test_zero_adapters_change_nothing():
    """A zero adapter gives the bits of a row without one."""
    from lightning_router.workloads import build_layer
    w = _workload(tokens=40, d_model=256, d_ff=512)
    layer, t = build_layer(w, device=DEV)
    layer.adapters = _adapters(layer, 2, 8, 4)
    for m in layer.adapters.mats:
        getattr(layer.adapters, f"{m}_b").zero_()
    none = torch.full((40,), -1, device=DEV)
    out, _ = layer(t.x, adapter_ids=none)
    assert torch.equal(layer(t.x, adapter_ids=none + 1)[0], out)
    ref, _ = layer(t.x)      # the fused epilogue: without the rounding of gate and up
    assert float((out.double() - ref.double()).norm() / ref.double().norm()) <= 1e-3


def test_load_pads_ranks():
    from lightning_router.models.adapters import ExpertAdapters
    ad = ExpertAdapters(2, 3, 64, 128, 16).to(DEV)
    A, B = torch.randn(5, 64), torch.randn(128, 5)
    ad.load(1, 2, "up", A, B, scale=0.25)
    bank = ad.bank("up")
    entry = 1 * 3 + 2
    assert torch.equal(bank.a[entry, :5].cpu(), A.half()) and not bank.a[entry, 5:].any()
    assert torch.equal(bank.b[entry, :, :5].cpu(), B.half()) and not bank.b[entry, :, 5:].any()
    assert bank.scale.tolist() == [1.0] * 5 + [0.25]
    for mat, a, b in (("side", A, B), ("up", torch.randn(17, 64), torch.randn(128, 17)),
                      ("down", A, B)):
        with pytest.raises(ValueError):
            ad.load(0, 0, mat, a, b)
    with pytest.raises(ValueError, match="rank"):
        ExpertAdapters(1, 1, 64, 64, 12)


def test_runner_serves_adapters():
    from lightning_router.serving.model_runner import LightningModelRunner
    from lightning_router.serving.worker import LightningRouterWorker
    from lightning_router.workloads import build_layer
    w = _workload(tokens=32, d_model=256, d_ff=512)
    layer, t = build_layer(w, device=DEV)
    cfg = (dict(hidden_size=256, intermediate_size=512),
           dict(num_experts=8, num_experts_per_token=2, expert_capacity_factor=1.25),
           dict(group_size=128), {})
    r = LightningModelRunner(*cfg, device="cuda:0")
    r.load_model()
    r.moe_layer.load_state_dict(layer.state_dict())
    r.set_adapters(_adapters(layer, 4, 8, 6))
    r.capture(32)
    r.capture(32, adapters=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(3):
        x = torch.randn(32, 256, generator=g, device=DEV).half()
        ids = torch.randint(-1, 4, (32,), generator=g, device=DEV)
        ref, _ = r.moe_layer(x, adapter_ids=ids)
        assert torch.equal(r.execute_model(None, x, adapter_ids=ids), ref)
        assert torch.equal(r.execute_model(None, x), r.moe_layer(x)[0])
        odd, _ = r.moe_layer(x[:20], adapter_ids=ids[:20])
        assert torch.equal(r.execute_model(None, x[:20], adapter_ids=ids[:20]), odd)
    with pytest.raises(ValueError, match="entries"):
        r.execute_model(None, x, adapter_ids=ids[:5])
    r.set_adapters(None)
    assert list(r._graphs) == [(32, 256)]
    with pytest.raises(RuntimeError, match="adapters is not set"):
        r.execute_model(None, x, adapter_ids=ids)
    wk = LightningRouterWorker(*cfg, serving_config={})
    wk.init_device()
    wk.load_model()
    wk.runner.moe_layer.load_state_dict(layer.state_dict())
    wk.runner.set_adapters(_adapters(layer, 4, 8, 6))
    ref, _ = wk.runner.moe_layer(x, adapter_ids=ids)
    assert torch.equal(wk.execute_model(None, x, adapter_ids=ids), ref)


def test_adapters_exchanged_behind_a_captured_graph():
    from lightning_router.serving.model_runner import LightningModelRunner
    from lightning_router.workloads import build_layer
    w = _workload(tokens=16, d_model=256, d_ff=512)
    layer, t = build_layer(w, device=DEV)
    r = LightningModelRunner(dict(hidden_size=256, intermediate_size=512),
                             dict(num_experts=8, num_experts_per_token=2), dict(group_size=128),
                             {}, device="cuda:0")
    r.load_model()
    r.moe_layer.load_state_dict(layer.state_dict())
    r.set_adapters(_adapters(layer, 4, 8, 6))
    r.capture(16, adapters=True)
    ids = torch.arange(16, device=DEV, dtype=torch.int32) % 4
    x = torch.randn(16, 256, device=DEV).half()
    old = r.execute_model(None, x, adapter_ids=ids)
    r.moe_layer.adapters = _adapters(layer, 4, 8, 7)      # not through set_adapters
    ref, _ = r.moe_layer(x, adapter_ids=ids)
    assert torch.equal(r.execute_model(None, x, adapter_ids=ids), ref)
    assert not torch.equal(old, ref)


def test_serving_with_adapters_takes_states_that_require_a_gradient():
    from lightning_router.workloads import build_layer
    layer, t = build_layer(_workload(tokens=16, d_model=256, d_ff=256), device=DEV)
    layer.adapters = _adapters(layer, 2, 8, 3)
    ids = torch.zeros(16, dtype=torch.int32, device=DEV)
    want, _ = layer(t.x, adapter_ids=ids)
    got, _ = layer(t.x.clone().requires_grad_(), adapter_ids=ids)
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# training
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [3, 64, 300, 3000])
def test_trainable_layer_has_the_same_output(tokens):
    from lightning_router.workloads import build_layer
    w = _workload("fine", tokens=tokens, d_model=256, d_ff=256)
    layer, t = build_layer(w, device=DEV)
    out, aux = layer(t.x)
    layer.trainable = True
    a, b = layer(t.x)
    assert a.requires_grad and b.requires_grad
    assert torch.equal(a.detach(), out)
    # the loss: the same probabilities, their sum over tokens in another order
    assert abs(float(b.detach()) - float(aux)) <= 2.0 ** -20 * float(aux)
    with torch.no_grad():
        assert torch.equal(layer(t.x)[0], out) and not layer(t.x)[0].requires_grad


def _weights64(x, W, bias, ids):
    logits = x.double() @ W.t()
    if bias is not None:
        logits = logits + bias.double()
    p = torch.softmax(logits, 1)
    ps = p.gather(1, ids)
    return p, ps / (ps.sum(1, keepdim=True) + 1e-9)


@pytest.mark.parametrize("with_adapters", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_router_gradient_over_frozen_experts(with_adapters, masked):
    """The whole step: INT4 experts (with adapters), combine, gate weight's gradient."""
    from lightning_router.kernels.routing_grad import dispatch_tokens
    from lightning_router.workloads import build_layer
    w = _workload("fine", tokens=500, d_model=256, d_ff=256, capacity_factor=0.8)
    layer, t = build_layer(w, device=DEV)
    layer.trainable = True
    layer.gate.gate_proj.float()                  # fp32 master weight
    g = torch.Generator(device=DEV).manual_seed(2)
    ids = None
    if with_adapters:
        layer.adapters = _adapters(layer, 3, 8, 9)
        ids = torch.randint(-1, 3, (500,), generator=g, device=DEV)
    mask = (torch.rand(500, generator=g, device=DEV) < 0.7) if masked else None
    G = torch.randn(500, 256, generator=g, device=DEV).half()
    out, aux = layer(t.x, adapter_ids=ids, token_mask=mask)
    ((out * G).float().sum() + 1000.0 * aux).backward()
    grad = layer.gate.gate_proj.weight.grad
    assert grad.dtype == torch.float32
    # 64-bit autograd over the same selection and the same (constant) expert rows
    with torch.no_grad():
        logits = layer.gate.differentiable_logits(t.x)
        plan = dispatch_tokens(t.x, logits, w.top_k, capacity=layer.capacity(500))
        y = layer.expert_forward(plan, ids).double()
    sel, pos = plan.expert_ids.view(500, -1).long(), plan.slot_pos.view(500, -1).long()
    W = layer.gate.gate_proj.weight.detach().half().double().requires_grad_()
    p, wts = _weights64(t.x, W, layer.gate.logit_bias, sel)
    rows = torch.where((pos >= 0)[..., None], y[pos.clamp(min=0)], 0.0)
    live = torch.ones(500, dtype=torch.bool, device=DEV) if mask is None else mask
    f = torch.bincount(sel[live].reshape(-1), minlength=w.experts).double() \
        / (int(live.sum()) * w.top_k)
    loss = ((wts[..., None] * rows).sum(1) * G.double()).sum() \
        + 1000.0 * layer.gate.load_balance_weight * w.experts * (f * p[live].mean(0)).sum()
    (want,) = torch.autograd.grad(loss, W)
    # fp32 throughout: sums of d = 256 and T = 500 products, softmax of 64: (256 + 500 + 96) U
    rel = float((grad.double() - want).norm() / want.norm())
    assert rel <= 852 * 2.0 ** -24 * 4, rel


def test_all_gradients_over_plain_experts():
    from lightning_router.config import KernelConfig, ModelConfig, MoEConfig, QuantizationConfig
    from lightning_router.models.moe_layer import MoELayer
    torch.manual_seed(0)
    T, d, f, E, k = 200, 64, 128, 4, 2
    layer = MoELayer(ModelConfig(hidden_size=d, intermediate_size=f),
                     MoEConfig(num_experts=E, num_experts_per_token=k, trainable=True,
                               expert_capacity_factor=0.9),
                     QuantizationConfig(enabled=False), KernelConfig()).cuda().half()
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(T, d, generator=g, device=DEV).half().requires_grad_()
    G = torch.randn(T, d, generator=g, device=DEV).half()
    out, aux = layer(x)
    ((out * G).float().sum() + 50.0 * aux).backward()
    with torch.no_grad():
        _, plan = layer.route(x.detach())
    sel, pos = plan.expert_ids.view(T, k).long(), plan.slot_pos.view(T, k).long()
    x64 = x.detach().double().requires_grad_()
    P = {n: p.detach().double().requires_grad_() for n, p in layer.named_parameters()}
    p, wts = _weights64(x64, P["gate.gate_proj.weight"], None, sel)
    o = torch.zeros(T, d, dtype=torch.float64, device=DEV)
    for e in range(E):
        tt, j = torch.nonzero((sel == e) & (pos >= 0), as_tuple=True)
        W = [P[f"experts.experts.{e}.{m}_proj.weight"] for m in ("gate", "up", "down")]
        xe = x64[tt]
        ye = (torch.nn.functional.silu(xe @ W[0].t()) * (xe @ W[1].t())) @ W[2].t()
        o = o.index_add(0, tt, ye * wts[tt, j][:, None])
    share = torch.bincount(sel.reshape(-1), minlength=E).double() / (T * k)
    loss = (o * G.double()).sum() + 50.0 * 0.01 * E * (share * p.mean(0)).sum()
    want = torch.autograd.grad(loss, [x64, *P.values()])
    # fp16 rows, products and gradients: about eight roundings of at most 2^-11 in a row
    for name, a, b in zip(["x", *P], [x.grad, *[q.grad for q in layer.parameters()]], want):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 8 * 2.0 ** -11, (name, rel)


def test_trainable_gate_module():
    from lightning_router.models.gating import TopKGating
    torch.manual_seed(1)
    gate = TopKGating(128, 8, 2, trainable=True).to(DEV)
    x = torch.randn(4, 25, 128, device=DEV, requires_grad=True)
    mask = torch.ones(100, dtype=torch.bool, device=DEV)
    mask[90:] = False
    ids, w, tok, aux = gate(x, token_mask=mask)
    assert tok.tolist() == [t for t in range(100) for _ in range(2)]
    (w.sum() * 0.0 + aux).backward()
    assert gate.gate_proj.weight.grad.abs().sum() > 0 and x.grad.abs().sum() > 0
    assert not x.grad.reshape(100, 128)[90:].any()
    with torch.no_grad():
        i2, w2, t2, a2 = gate(x)
    assert torch.equal(ids, i2) and torch.equal(tok, t2)
    with pytest.raises(ValueError, match="token_mask"), torch.no_grad():
        gate(x, token_mask=mask)


def test_a_few_steps_of_router_training():
    """Router tuning over INT4 experts with adapters, as a user runs it."""
    from lightning_router.workloads import build_layer
    w = _workload("fine", tokens=256, d_model=256, d_ff=256)
    layer, t = build_layer(w, device=DEV)
    layer.trainable = True
    layer.gate.gate_proj.float()
    layer.adapters = _adapters(layer, 2, 8, 1)
    ids = (torch.arange(256, device=DEV) // 128)
    target = torch.randn(256, 256, device=DEV)
    opt = torch.optim.SGD([layer.gate.gate_proj.weight], lr=1e-3)
    seen = []
    for _ in range(4):
        out, aux = layer(t.x, adapter_ids=ids)
        loss = ((out.float() - target) ** 2).mean() * 1024 + 1024 * aux   # fp16 gradients
        opt.zero_grad()
        loss.backward()
        seen.append(layer.gate.gate_proj.weight.grad.clone())
        opt.step()
    assert all(torch.isfinite(s).all() and s.abs().sum() > 0 for s in seen)
    assert not torch.equal(seen[0], seen[-1])


def test_refusals():
    from lightning_router.workloads import build_layer
    w = _workload(tokens=16, d_model=256, d_ff=256)
    layer, t = build_layer(w, device=DEV)
    ids = torch.zeros(16, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="adapters is not set"):
        layer(t.x, adapter_ids=ids)
    with pytest.raises(ValueError, match="entries"):
        layer(t.x, adapter_ids=ids[:3])
    with pytest.raises(ValueError, match="token_mask"):
        layer(t.x, token_mask=ids == 0)
    layer.trainable = True
    with pytest.raises(RuntimeError, match="frozen"):
        layer(t.x.clone().requires_grad_())

"""Cases of the operators that adapt the MoE layer: the router's training path and low-rank adapters.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same ranges, ``prepare(case, seed)``
makes the inputs on the GPU, ``run(state)`` is one pass, ``work(case)`` the bytes and operations it cannot
do without and ``exact(case, seed)`` its outputs in 64 bits.  With ``own`` false a pass is the operators'
plain form (elementary torch operations in 32 bits, one rounding at the end); with ``own`` true it makes the
framework's calls.

The operators (``op``):

``gating``    top-k softmax weights, per-expert counts and the balance loss from fp32 logits, with the
              gradient of weights and loss in the logits.
``gate``      the gate projection h W^T + b with its gradients in h, W and b.
``route``     dispatch of token rows to experts under a capacity, and the weighted combine of the experts'
              rows, with the gradients in the tokens, the logits and the experts' rows.
``adapters``  low-rank adapters of many requests beside a shared projection's output (form ``add``), or
              beside a SwiGLU expert's gate and up projections with one adapter per (request, expert)
              (form ``swiglu``).
"""

import math
import sys
from pathlib import Path

import torch

own = False

LBW = 0.01
EPS = 1e-9


def _package():
    """The framework's modules, imported once (its package directory goes on sys.path, as for any user)."""
    if not hasattr(_package, "modules"):
        where = str(Path(__file__).resolve().parents[1] / "llm-serving-kernel-optimization_b200")
        if where not in sys.path:
            sys.path.insert(0, where)
        from lightning_router.kernels import adapters, routing_grad
        _package.modules = adapters, routing_grad
    return _package.modules


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a micro-batch of a small router (the 4-expert default configuration): latency counts
        dict(name="gating_1k_e4", op="gating", tokens=1000, experts=4, top_k=2, padded=0.0),
        # the fine-grained layer's training batch, a fifth of it padding
        dict(name="gating_8k_e64_padded", op="gating", tokens=8192, experts=64, top_k=6, padded=0.2),
        # the largest batch of the dispatch sweep
        dict(name="gating_262k_e8", op="gating", tokens=262144, experts=8, top_k=2, padded=0.0),
        # router training at the prefill batch of the 8-expert layer
        dict(name="gate_16k_e8", op="gate", tokens=16384, d_model=4096, experts=8),
        # router training of the fine-grained layer, a ragged batch
        dict(name="gate_8k_e64_ragged", op="gate", tokens=8111, d_model=2048, experts=64),
        # the routing path of a training step at the prefill batch
        dict(name="route_16k_e8", op="route", tokens=16384, d_model=4096, experts=8, top_k=2,
             capacity_factor=1.25),
        # a small ragged batch of the fine-grained layer with many dropped slots
        dict(name="route_777_e64_drops", op="route", tokens=777, d_model=2048, experts=64, top_k=6,
             capacity_factor=0.5),
        # one user's decode step on a square projection: latency counts
        dict(name="adapters_1_token", op="adapters", form="add", tokens=1, requests=1, d_in=4096,
             d_out=4096, adapters=4, rank=8, without=0.0),
        # a decode batch, every request with an adapter of its own
        dict(name="adapters_decode64", op="adapters", form="add", tokens=64, requests=64, d_in=4096,
             d_out=14336, adapters=64, rank=16, without=0.0),
        # chunks of a few requests' prompts in one ragged batch, some requests without an adapter
        dict(name="adapters_ragged", op="adapters", form="add", tokens=1111, requests=9, d_in=2048,
             d_out=1408, adapters=6, rank=64, without=0.3),
        # the prefill batch beside the up projection
        dict(name="adapters_prefill16k", op="adapters", form="add", tokens=16384, requests=8,
             d_in=4096, d_out=14336, adapters=8, rank=32, without=0.0),
        # a decode batch inside the MoE layer: 64 tokens x 2 experts, 8 adapters on each of 8 experts
        dict(name="adapters_experts_decode", op="adapters", form="swiglu", tokens=128, requests=64,
             d_in=4096, d_out=14336, adapters=64, rank=16, without=0.1),
    ]


def _log(rng, low, high, step=1):
    """A multiple of `step` between low and high, even over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + step)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    op = rng.choice(["gating", "gate", "route", "adapters", "adapters"])
    if op == "gating":
        experts = rng.randint(2, 64)
        return dict(op=op, tokens=_log(rng, 1, 262144 * 8 // max(8, experts)), experts=experts,
                    top_k=rng.randint(1, min(experts, 8)), padded=rng.choice([0.0, 0.1, 0.5]))
    if op == "gate":
        return dict(op=op, tokens=_log(rng, 1, 16384), d_model=_log(rng, 64, 4096, 16),
                    experts=rng.randint(2, 64))
    if op == "route":
        experts = rng.randint(2, 64)
        top_k = rng.randint(1, min(experts, 8))
        d = _log(rng, 64, 4096, 8)
        most = min(16384, 16384 * 2 * 4096 // (top_k * d))
        return dict(op=op, tokens=_log(rng, 1, most), d_model=d, experts=experts, top_k=top_k,
                    capacity_factor=rng.choice([0.5, 1.0, 1.25, 2.0]))
    n = _log(rng, 1, 64)
    rank = rng.choice([8, 16, 24, 32, 64, 128])
    k, f = _log(rng, 64, 4096, 8), _log(rng, 64, 14336, 8)
    form = rng.choice(["add", "add", "swiglu"])
    # the plain form multiplies every row with every adapter: no more of that than in the largest listed case
    most = int(min(16384, 16384 * 8 * 32 / (n * rank * (2 if form == "swiglu" else 1))))
    tokens = _log(rng, 1, max(1, most))
    return dict(op=op, form=form, tokens=tokens, requests=min(tokens, _log(rng, 1, 64)), d_in=k,
                d_out=f, adapters=n, rank=rank, without=rng.choice([0.0, 0.2]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    c = case
    s = dict(c)
    if c["op"] == "gating":
        T, E, k = c["tokens"], c["experts"], c["top_k"]
        s["logits"] = _normal(g, T, E).requires_grad_()
        s["mask"] = (torch.rand(T, generator=g, device="cuda") >= c["padded"]) if c["padded"] else None
        # gradients of a loss averaged over the tokens
        s["d_weights"] = _normal(g, T * k, std=1.0 / T)
        s["d_aux"] = torch.ones((), device="cuda")
    elif c["op"] == "gate":
        T, d, E = c["tokens"], c["d_model"], c["experts"]
        s["h"] = _normal(g, T, d, dtype=torch.float16).requires_grad_()
        s["weight"] = _normal(g, E, d, std=0.02).requires_grad_()     # fp32 master weight
        s["bias"] = _normal(g, E, std=0.1).requires_grad_()
        s["d_logits"] = _normal(g, T, E, std=0.1)
    elif c["op"] == "route":
        T, d, E, k = c["tokens"], c["d_model"], c["experts"], c["top_k"]
        s["x"] = _normal(g, T, d, dtype=torch.float16).requires_grad_()
        s["logits"] = _normal(g, T, E).requires_grad_()
        s["y"] = _normal(g, T * k, d, dtype=torch.float16).requires_grad_()   # the experts' rows
        # fp16 gradients under a loss scale of T
        s["d_out"] = _normal(g, T, d, std=0.1, dtype=torch.float16)
        s["d_permuted"] = _normal(g, T * k, d, std=0.1, dtype=torch.float16)
        s["d_aux"] = torch.full((), float(T), device="cuda")
    else:
        T, K, N, n, r = c["tokens"], c["d_in"], c["d_out"], c["adapters"], c["rank"]
        R = c["requests"]
        s["x"] = _normal(g, T, K, dtype=torch.float16)
        # contiguous requests of ragged lengths (one token each in a decode batch)
        if R < T:
            cuts = torch.randperm(T - 1, generator=g, device="cuda")[:R - 1].sort().values + 1
        else:
            cuts = torch.arange(1, T, device="cuda")
        request = torch.searchsorted(cuts, torch.arange(T, device="cuda"), right=True)
        adapter = torch.arange(R, device="cuda") % n
        adapter = adapter[torch.randperm(R, generator=g, device="cuda")]
        adapter[torch.rand(R, generator=g, device="cuda") < c["without"]] = -1
        s["index"] = adapter[request].to(torch.int32)
        names = ("gate", "up") if c["form"] == "swiglu" else ("base",)
        for m in names:
            s[m] = _normal(g, T, N, dtype=torch.float16)
            s[m + "_a"] = _normal(g, n, r, K, std=K ** -0.5, dtype=torch.float16)
            s[m + "_b"] = _normal(g, n, N, r, std=0.1, dtype=torch.float16)
            s[m + "_scale"] = torch.rand(n, generator=g, device="cuda") + 0.5
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"gating": _gating, "gate": _gate, "route": _route, "adapters": _adapters}[s["op"]](s)


def _run_own(s):
    adapters, routing_grad = _package()
    if s["op"] == "gating":
        g = routing_grad.balanced_gating(s["logits"], s["top_k"], LBW, token_mask=s["mask"])
        (dl,) = torch.autograd.grad((g.gate_weights, g.aux_loss), (s["logits"],),
                                    (s["d_weights"], s["d_aux"]))
        return dict(ids=g.expert_ids, weights=g.gate_weights, counts=g.expert_counts, aux=g.aux_loss,
                    d_logits=dl)
    if s["op"] == "gate":
        logits = routing_grad.gate_projection(s["h"], s["weight"], s["bias"])
        dh, dw, db = torch.autograd.grad((logits,), (s["h"], s["weight"], s["bias"]), (s["d_logits"],))
        return dict(logits=logits, d_h=dh, d_weight=dw, d_bias=db)
    if s["op"] == "route":
        plan = routing_grad.dispatch_tokens(s["x"], s["logits"], s["top_k"], s["capacity_factor"], LBW)
        out = routing_grad.combine_tokens(s["y"], plan.gate_weights, plan)
        dx, dl, dy = torch.autograd.grad((out, plan.permuted, plan.aux_loss),
                                         (s["x"], s["logits"], s["y"]),
                                         (s["d_out"], s["d_permuted"], s["d_aux"]))
        return dict(permuted=plan.permuted, out=out, aux=plan.aux_loss, d_x=dx, d_logits=dl, d_y=dy)
    if s["form"] == "add":
        bank = adapters.AdapterBank(s["base_a"], s["base_b"], s["base_scale"])
        return adapters.adapter_add(s["base"], s["x"], bank, s["index"])
    gate = adapters.AdapterBank(s["gate_a"], s["gate_b"], s["gate_scale"])
    up = adapters.AdapterBank(s["up_a"], s["up_b"], s["up_scale"])
    return adapters.adapter_swiglu(s["gate"], s["up"], s["x"], gate, up, s["index"])


def _top_k(logits, k):
    """Softmax, the k largest logits' experts (ties: lowest first) and their normalised weights."""
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = p.gather(1, ids)
    q = chosen.sum(1, keepdim=True) + EPS
    return p, ids, chosen / q, q


def _logit_gradient(p, ids, w, q, d_w, d_p):
    """d_p plus the weights' gradient, taken back through the softmax."""
    d_p = d_p.scatter_add(1, ids, (d_w - (d_w * w).sum(1, keepdim=True)) / q)
    return p * (d_p - (p * d_p).sum(1, keepdim=True))


def _gating(s):
    logits, k = s["logits"].detach(), s["top_k"]
    T, E = logits.shape
    live = torch.ones(T, device=logits.device) if s["mask"] is None else s["mask"].float()
    p, ids, w, q = _top_k(logits, k)
    w = w * live[:, None]
    n = live.sum().clamp(min=1.0)
    counts = (torch.nn.functional.one_hot(ids, E).sum(1) * live[:, None].long()).sum(0)
    f = counts.float() / (n * k)
    mean_p = ((p * live[:, None]).sum(0, dtype=torch.float64) / n).float()
    aux = LBW * E * (f * mean_p).sum()
    d_p = (s["d_aux"] * LBW * E * f / n)[None, :].expand(T, E)
    dl = _logit_gradient(p, ids, w, q, s["d_weights"].view(T, k), d_p) * live[:, None]
    return dict(ids=ids.reshape(-1).int(), weights=w.reshape(-1), counts=counts.int(), aux=aux,
                d_logits=dl)


def _gate(s):
    h = s["h"].detach().float()
    w = s["weight"].detach().half().float()     # the projection's weight is fp16
    dl = s["d_logits"]
    return dict(logits=h @ w.t() + s["bias"].detach(), d_h=(dl @ w).half(), d_weight=dl.t() @ h,
                d_bias=dl.sum(0))


def _route(s):
    x, logits, y = s["x"].detach(), s["logits"].detach(), s["y"].detach()
    k, d_out, d_perm = s["top_k"], s["d_out"].float(), s["d_permuted"].float()
    T, E = logits.shape
    S = T * k
    p, ids, w, q = _top_k(logits, k)
    capacity = max(int((S / E) * s["capacity_factor"]), 1)
    flat = ids.reshape(-1)
    hot = torch.nn.functional.one_hot(flat, E)
    rank = (hot.cumsum(0) - hot).gather(1, flat[:, None])[:, 0]
    counts = hot.sum(0)
    row = (counts.cumsum(0) - counts)[flat] + rank          # the row of each slot
    kept = (rank < capacity).float()
    slot = torch.empty_like(row)
    slot[row] = torch.arange(S, device=row.device)          # the slot of each row
    token, row_kept = slot // k, kept[slot][:, None]
    permuted = (x[token].float() * row_kept).half()
    f = counts.float() / S
    aux = LBW * E * (f * p.sum(0, dtype=torch.float64).float() / T).sum()
    wk = w.reshape(-1) * kept
    rows = y[row].float().view(T, k, -1)
    out = (rows * wk.view(T, k, 1)).sum(1).half()
    d_w = (rows * d_out[:, None, :]).sum(2) * kept.view(T, k)
    d_y = (d_out[token] * wk[slot][:, None]).half()
    d_x = (d_perm[row] * kept[:, None]).view(T, k, -1).sum(1).half()
    d_p = (s["d_aux"] * LBW * E * f / T)[None, :].expand(T, E)
    return dict(permuted=permuted, out=out, aux=aux, d_x=d_x,
                d_logits=_logit_gradient(p, ids, w, q, d_w, d_p), d_y=d_y)


def _low_rank(x, a, b, scale, index):
    """scale (x A^T) B^T by each row's adapter: every adapter's product, kept where the row has it."""
    n, r, K = a.shape
    has = (index[:, None] == torch.arange(n, device=index.device)).float() * scale
    v = (x.float() @ a.float().view(n * r, K).t()).view(-1, n, r) * has[:, :, None]
    return v.view(-1, n * r) @ b.float().transpose(1, 2).reshape(n * r, -1)


def _adapters(s):
    if s["form"] == "add":
        return (s["base"].float() + _low_rank(s["x"], s["base_a"], s["base_b"], s["base_scale"],
                                              s["index"])).half()
    g = s["gate"].float() + _low_rank(s["x"], s["gate_a"], s["gate_b"], s["gate_scale"], s["index"])
    u = s["up"].float() + _low_rank(s["x"], s["up_a"], s["up_b"], s["up_scale"], s["index"])
    return (g / (1.0 + torch.exp(-g)) * u).half()


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    T = c["tokens"]
    if c["op"] == "gating":
        E, S = c["experts"], T * c["top_k"]
        # logits forward and backward, their gradient; ids and weights out, the weights' gradient in
        return dict(bytes=12 * T * E + 12 * S + (T if c["padded"] else 0), flops=30 * T * E)
    if c["op"] == "gate":
        d, E = c["d_model"], c["experts"]
        # the rows forward, the rows for the weight's gradient, the rows' gradient; logits and theirs
        return dict(bytes=6 * T * d + 8 * T * E + 8 * E * d, flops=6 * T * d * E)
    if c["op"] == "route":
        d, E, k = c["d_model"], c["experts"], c["top_k"]
        S = T * k
        kept = min(S, E * max(int(S / E * c["capacity_factor"]), 1))
        # forward: x in, permuted out, kept y in, out out; backward: d_out in, kept y in, d_y out,
        # kept d_permuted in, d_x out; the logits twice and their gradient
        return dict(bytes=2 * d * (4 * T + 3 * kept + 2 * S) + 12 * T * E + 24 * S,
                    flops=8 * kept * d)
    K, N, r = c["d_in"], c["d_out"], c["rank"]
    m = 2 if c["form"] == "swiglu" else 1
    live = min(c["adapters"], max(1, round(c["requests"] * (1 - c["without"]))))
    return dict(bytes=2 * T * (K + (m + 1) * N) + 2 * m * live * r * (K + N) + 4 * T,
                flops=2 * T * m * r * (K + N))


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    with torch.no_grad():
        return {"gating": _exact_gating, "gate": _exact_gate, "route": _exact_route,
                "adapters": _exact_adapters}[case["op"]](s)


def _exact_choice(logits, k):
    order = torch.argsort(-logits, dim=1, stable=True)[:, :k]
    z = logits.double()
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    return order, p


def _exact_back(p, order, d_w, d_p):
    """The gradient in the logits from the Jacobians of the weights and of the softmax."""
    T, k = order.shape
    ps = torch.gather(p, 1, order)
    q = ps.sum(1) + EPS
    # w_j = ps_j / q: dw_j/dps_i = [i == j]/q - ps_j/q^2
    d_ps = d_w / q[:, None] - ((d_w * ps).sum(1) / q ** 2)[:, None]
    grad = d_p.clone()
    for j in range(k):
        col = order[:, j]
        grad[torch.arange(T, device=p.device), col] += d_ps[:, j]
    return p * grad - p * (p * grad).sum(1, keepdim=True)


def _exact_gating(s):
    logits, k = s["logits"], s["top_k"]
    T, E = logits.shape
    live = torch.ones(T, dtype=torch.bool, device=logits.device) if s["mask"] is None else s["mask"]
    n = max(int(live.sum()), 1)
    order, p = _exact_choice(logits, k)
    w = torch.gather(p, 1, order)
    w = w / (w.sum(1, keepdim=True) + EPS)
    w[~live] = 0.0
    counts = torch.bincount(order[live].reshape(-1), minlength=E)
    share = counts.double() / (n * k)
    aux = LBW * E * torch.dot(share, p[live].sum(0) / n)
    d_p = (share * (float(s["d_aux"]) * LBW * E / n)).repeat(T, 1)
    dl = _exact_back(p, order, s["d_weights"].double().reshape(T, k), d_p)
    dl[~live] = 0.0
    return dict(ids=None, weights=w.reshape(-1), counts=None, aux=aux, d_logits=dl)


def _exact_gate(s):
    h, dl = s["h"].double(), s["d_logits"].double()
    w = s["weight"].half().double()
    return dict(logits=torch.einsum("td,ed->te", h, w) + s["bias"].double(),
                d_h=torch.einsum("te,ed->td", dl, w), d_weight=torch.einsum("te,td->ed", dl, h),
                d_bias=dl.sum(0))


def _exact_route(s):
    x, logits, y, k = s["x"], s["logits"], s["y"], s["top_k"]
    T, E = logits.shape
    S, d = T * k, x.shape[1]
    cap = max(int((S / E) * s["capacity_factor"]), 1)
    order, p = _exact_choice(logits, k)
    w = torch.gather(p, 1, order)
    w = (w / (w.sum(1, keepdim=True) + EPS)).reshape(-1)
    flat = order.reshape(-1)
    counts = torch.bincount(flat, minlength=E)
    out = torch.zeros(T, d, dtype=torch.float64, device=x.device)
    d_x, d_y = torch.zeros_like(out), torch.zeros(S, d, dtype=torch.float64, device=x.device)
    d_w = torch.zeros(S, dtype=torch.float64, device=x.device)
    permuted = torch.zeros(S, d, dtype=torch.float64, device=x.device)
    first = 0
    for e in range(E):
        slots = torch.nonzero(flat == e)[:, 0][:cap]        # the expert's kept slots, in slot order
        rows = slice(first, first + slots.numel())
        first += int(counts[e])
        t = slots // k
        permuted[rows] = x[t].double()
        ye, de = y[rows].double(), s["d_out"][t].double()
        out.index_add_(0, t, ye * w[slots, None])
        d_x.index_add_(0, t, s["d_permuted"][rows].double())
        d_y[rows] = de * w[slots, None]
        d_w[slots] = (de * ye).sum(1)
    share = counts.double() / S
    aux = LBW * E * torch.dot(share, p.mean(0))
    d_p = (share * (float(s["d_aux"]) * LBW * E / T)).repeat(T, 1)
    return dict(permuted=permuted, out=out, aux=aux, d_x=d_x,
                d_logits=_exact_back(p, order, d_w.reshape(T, k), d_p), d_y=d_y)


def _exact_adapters(s):
    def product(base, a, b, scale):
        o = base.double()
        for i in range(a.shape[0]):
            t = torch.nonzero(s["index"] == i)[:, 0]
            if t.numel():
                v = torch.mm(s["x"][t].double(), a[i].double().t())
                o[t] += float(scale[i]) * torch.mm(v, b[i].double().t())
        return o

    if s["form"] == "add":
        return product(s["base"], s["base_a"], s["base_b"], s["base_scale"])
    g = product(s["gate"], s["gate_a"], s["gate_b"], s["gate_scale"])
    return g * torch.sigmoid(g) * product(s["up"], s["up_a"], s["up_b"], s["up_scale"])

"""Mixture-of-Experts layer, reference ``lightning_router/models/moe_layer.py:20-135``.

``MoELayer(model_cfg, moe_cfg, quant_cfg, kernel_cfg).forward(h) -> (out, aux_loss)``
with ``h`` of shape (B, S, d) or (T, d).  One forward is six stream-ordered
launches and no host synchronisation:

1. gate projection             fp16 h . fp16 Wg^T -> fp32 logits        (CUDA cores / mma.sync)
2. top-k softmax + histogram   ids, weights, slot ranks, aux loss, CSR offsets
   (up to 256 tokens, 1 and 2 are one launch: the decode step is five)
3. permute                     token rows -> expert-contiguous rows (kept slots only)
4. grouped W4A16 gate/up GEMM  tcgen05, fused SwiGLU (or SiLU) epilogue
5. grouped W4A16 down GEMM     tcgen05
6. combine                     token-major fp32 weighted sum, one fp16 store

Capacity is ``max(int(T*k/E * cf), 1)`` per expert (reference
``expert_routing.py:196-197``); slots beyond it are dropped in slot order.
``routing_implementation`` is accepted for configuration compatibility; there
is a single (CUDA) implementation.

Two optional uses:

* **adapters**: with ``layer.adapters`` (:class:`ExpertAdapters`) set,
  ``forward(h, adapter_ids=ids)`` adds each token's low-rank adapter to its
  experts' projections (INT4 experts); tokens with id -1 go without.  A call with
  ids leaves the fused SwiGLU product for all tokens (gate and up are written,
  rounded to fp16, and read again), also where every id is -1: pass ``None`` then.
* **training** (``MoEConfig.trainable``, gradients enabled): the output and the
  balance loss carry gradients.  INT4 experts are frozen: the router's weight
  learns from their rows, which are constants, and hidden states must not
  require a gradient.  With a ``token_mask`` the loss is :func:`balanced_gating`'s.
  Plain experts (``QuantizationConfig(enabled=False)``)
  train with the router, gradients reach the hidden states.  Row gradients are
  fp16: scale the loss.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from lightning_router.config import KernelConfig, ModelConfig, MoEConfig, QuantizationConfig
from lightning_router.kernels.adapters import adapter_rows
from lightning_router.kernels.expert_routing import (
    SMALL_BATCH_TOKENS, RoutingPlan, combine, expert_capacity, gate_topk_gating_dispatch,
    topk_gating_dispatch)
from lightning_router.kernels.routing_grad import (
    DispatchPlan, balanced_gating, combine_tokens, dispatch_tokens)
from lightning_router.models.experts import ExpertGroup
from lightning_router.models.gating import TopKGating


class MoELayer(nn.Module):
    def __init__(self, model_cfg: ModelConfig, moe_cfg: MoEConfig,
                 quant_cfg: QuantizationConfig, kernel_cfg: KernelConfig):
        super().__init__()
        self.moe_cfg = moe_cfg
        self.kernel_cfg = kernel_cfg
        self.hidden_size = model_cfg.hidden_size
        self.intermediate_size = model_cfg.intermediate_size
        self.num_experts = moe_cfg.num_experts
        self.top_k = moe_cfg.num_experts_per_token
        self.gate = TopKGating(
            hidden_size=model_cfg.hidden_size,
            num_experts=moe_cfg.num_experts,
            top_k=moe_cfg.num_experts_per_token,
            load_balance_weight=moe_cfg.load_balance_loss_weight,
            bias=getattr(moe_cfg, "gate_bias", False),
            trainable=getattr(moe_cfg, "trainable", False),
        )
        self.trainable = getattr(moe_cfg, "trainable", False)
        self.experts = ExpertGroup(
            num_experts=moe_cfg.num_experts,
            hidden_size=model_cfg.hidden_size,
            intermediate_size=model_cfg.intermediate_size,
            quantized=quant_cfg.enabled and quant_cfg.quantize_experts,
            group_size=quant_cfg.group_size,
            activation=getattr(moe_cfg, "expert_activation", "swiglu"),
        )

        self.adapters = None   # an ExpertAdapters module, when adapters are served
        # optional list; when set, each forward appends (stage, cuda.Event) marks
        self.stage_events: list | None = None

    def _mark(self, name: str) -> None:
        if self.stage_events is not None:
            ev = torch.cuda.Event(enable_timing=True)
            ev.record()
            self.stage_events.append((name, ev))

    def capacity(self, num_tokens: int) -> int:
        return expert_capacity(num_tokens * self.top_k, self.num_experts,
                               self.moe_cfg.expert_capacity_factor)

    def route(self, hidden_states: torch.Tensor) -> tuple[torch.Tensor, RoutingPlan]:
        """Gate logits and the dispatch plan (rows permuted) for (T, d) fp16 input."""
        if hidden_states.shape[0] <= SMALL_BATCH_TOKENS:
            # decode-sized batches: projection, top-k and routing in one launch
            logits, plan = gate_topk_gating_dispatch(
                hidden_states, self.gate.gate_proj.weight.detach(), self.gate.logit_bias,
                self.top_k, load_balance_weight=self.gate.load_balance_weight,
                capacity=self.capacity(hidden_states.shape[0]))
            self._mark("gate")
            return logits, plan
        logits = self.gate.logits(hidden_states)
        self._mark("gate")
        plan = topk_gating_dispatch(hidden_states, logits, self.top_k,
                                    load_balance_weight=self.gate.load_balance_weight,
                                    capacity=self.capacity(hidden_states.shape[0]))
        return logits, plan

    def expert_forward(self, plan: RoutingPlan | DispatchPlan,
                       adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
        """Expert outputs for the kept rows of ``plan.permuted``."""
        if adapter_ids is not None:
            if self.adapters is None:
                raise RuntimeError("adapter_ids given, but layer.adapters is not set")
            if not self.experts.quantized:
                raise RuntimeError("adapters are served beside INT4 experts only")
            self.adapters.check(self.experts)
            with torch.no_grad():   # as without adapters, the experts build no graph
                index = adapter_rows(adapter_ids, plan, self.adapters.num_adapters)
                return self.experts.forward_segments_adapted(
                    plan.permuted, plan.offsets[:-1], plan.kept_counts, plan.capacity,
                    self.adapters, index, mark=self._mark)
        if self.experts.quantized:
            seg_start = plan.offsets[:-1]
            return self.experts.forward_segments(plan.permuted, seg_start, plan.kept_counts,
                                                 plan.capacity, mark=self._mark)
        # unquantized experts (reference nn.Linear path): per-expert slices
        y = torch.zeros_like(plan.permuted)
        offs = plan.offsets.tolist()
        kept = plan.kept_counts.tolist()
        for e, ex in enumerate(self.experts.experts):
            if kept[e]:
                rows = slice(offs[e], offs[e] + kept[e])
                y[rows] = ex(plan.permuted[rows]).to(y.dtype)
        return y

    def _differentiable_experts(self, plan: DispatchPlan) -> torch.Tensor:
        """Plain experts over the plan's segments; rows of dropped slots are zero."""
        sizes = plan.offsets.diff().tolist()
        kept = plan.kept_counts.tolist()
        rows = []
        for ex, seg, n in zip(self.experts.experts, plan.permuted.split(sizes), kept):
            if n:
                rows.append(ex(seg[:n]).to(torch.float16))
            if n < seg.shape[0]:
                rows.append(torch.zeros_like(seg[n:]))
        return torch.cat(rows)

    def _training_forward(self, hidden_states, adapter_ids, token_mask):
        h = hidden_states.reshape(-1, hidden_states.shape[-1])
        frozen = self.experts.quantized
        if frozen and hidden_states.requires_grad:
            raise RuntimeError("INT4 experts are frozen and give their rows no gradient: detach "
                               "the hidden states to train the router, or use plain experts")
        if adapter_ids is not None and not frozen:
            raise RuntimeError("adapters are served beside INT4 experts only")
        h = h.to(torch.float16)
        logits = self.gate.differentiable_logits(h)
        plan = dispatch_tokens(h, logits, self.top_k,
                               load_balance_weight=self.gate.load_balance_weight,
                               capacity=self.capacity(h.shape[0]))
        if frozen:
            with torch.no_grad():
                y = self.expert_forward(plan, adapter_ids)
        else:
            y = self._differentiable_experts(plan)
        out = combine_tokens(y, plan.gate_weights, plan)
        aux = plan.aux_loss if token_mask is None else balanced_gating(
            logits, self.top_k, self.gate.load_balance_weight,
            token_mask.reshape(-1)).aux_loss
        return out.to(hidden_states.dtype).view(hidden_states.shape), aux

    def forward(self, hidden_states: torch.Tensor, adapter_ids: torch.Tensor | None = None,
                token_mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """``adapter_ids``: an adapter number per token (any shape with T entries), -1 for
        none.  ``token_mask`` (training only): tokens that enter the balance loss."""
        if adapter_ids is not None and \
                adapter_ids.numel() != hidden_states.numel() // hidden_states.shape[-1]:
            raise ValueError(f"adapter_ids has {adapter_ids.numel()} entries for "
                             f"{hidden_states.numel() // hidden_states.shape[-1]} tokens")
        if self.trainable and torch.is_grad_enabled():
            return self._training_forward(hidden_states, adapter_ids, token_mask)
        if token_mask is not None:
            raise ValueError("token_mask needs a trainable layer with gradients enabled")
        orig_shape, orig_dtype = hidden_states.shape, hidden_states.dtype
        h = hidden_states.reshape(-1, orig_shape[-1]).to(torch.float16).contiguous()
        T = h.shape[0]
        self._mark("begin")
        _logits, plan = self.route(h)
        self._mark("dispatch")
        y = self.expert_forward(plan, adapter_ids)
        out = combine(y, plan.gate_weights, plan.slot_pos, T, self.top_k)
        self._mark("combine")
        return out.to(orig_dtype).view(orig_shape), plan.aux_loss

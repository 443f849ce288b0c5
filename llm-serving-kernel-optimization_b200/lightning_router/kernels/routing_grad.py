"""The routing path with gradients: train the router, over frozen INT4 experts or with plain ones.

Differentiable counterparts of the functions in :mod:`lightning_router.kernels.expert_routing`.
``gate_projection``, ``dispatch_tokens`` and ``combine_tokens`` give the inference functions' bits.
``balanced_gating`` selects the same experts, except that a NaN logit of a live token comes last
here and is taken by the inference scan where it leads; its weights and loss may differ in the
last bits (sums in another order).  The backward passes are sm_100a kernels without atomics (the
same inputs give the same bits).

* :func:`balanced_gating` -- top-k softmax weights, per-expert counts and the balance loss
  from logits, without a dispatch; a token mask keeps padding out.
* :func:`gate_projection` -- :func:`gate_logits` with gradients for the hidden rows, the
  weight (also an fp32 master weight) and the bias.
* :func:`dispatch_tokens` -- :func:`topk_gating_dispatch` whose plan carries gradients:
  ``permuted`` to ``x``, ``gate_weights`` and ``aux_loss`` to ``logits``.
* :func:`combine_tokens` -- :func:`combine` with gradients for the experts' rows and the weights.

Gradients follow the formulas of a loss in which the selection and the slot counts are
constants, as in the Switch balance loss.  Gradients of fp16 rows are fp16: scale the loss so
that they stay in range.  The gate's gradient of fp32 or bf16 hidden rows is rounded to their
type alone.  Logit, weight and bias gradients are fp32.  Each function is differentiable once
(``create_graph=True`` raises).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from lightning_router import _ext
from lightning_router.kernels.expert_routing import expert_capacity


class BalancedGating(NamedTuple):
    expert_ids: torch.Tensor      # (S,) int32, slot s = t * k + j
    gate_weights: torch.Tensor    # (S,) fp32, 0 for padded tokens
    expert_counts: torch.Tensor   # (E,) int32, slots of live tokens per expert
    aux_loss: torch.Tensor        # () fp32


class DispatchPlan(NamedTuple):
    """:class:`RoutingPlan` (same fields, same order) and the top-k it was made with."""
    expert_ids: torch.Tensor
    gate_weights: torch.Tensor
    token_indices: torch.Tensor
    offsets: torch.Tensor
    kept_counts: torch.Tensor
    aux_loss: torch.Tensor
    permuted: torch.Tensor
    routing_weights: torch.Tensor
    source_indices: torch.Tensor
    slot_pos: torch.Tensor
    capacity: int
    top_k: int


def balanced_gating(logits: torch.Tensor, top_k: int, load_balance_weight: float = 0.01,
                    token_mask: torch.Tensor | None = None) -> BalancedGating:
    """Top-k gating with the balance loss from fp32 ``logits`` (T, E), differentiable in them.

    ``aux_loss = lbw * E * sum_e f_e P_e`` over the live tokens (``token_mask`` (T,) bool,
    ``None``: all), ``f_e`` the share of their slots on expert e and ``P_e`` their mean
    probability.  A padded token has valid ids, weight 0, no part in counts or loss and a
    zero gradient, whatever its logits hold.  ``E <= 64``, ``top_k <= min(E, 8)``; T may be 0.
    """
    _ext.require_cuda(logits, token_mask)
    return BalancedGating(*_ext.ops().balanced_gating(logits.float(), token_mask, int(top_k),
                                                      float(load_balance_weight)))


def gate_projection(hidden: torch.Tensor, gate_weight: torch.Tensor,
                    bias: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 logits ``hidden @ gate_weight.T (+ bias)`` from operands rounded to fp16,
    differentiable in all three.  ``hidden`` (T, d) and ``gate_weight`` (E, d) of any
    floating type (a gradient has its tensor's type, rounded once from fp32 sums);
    ``d % 16 == 0``, ``E <= 256``.  As in any product, a hidden row that is not finite leaves
    the weight's gradient not finite, also where the row's own logits have no gradient."""
    _ext.require_cuda(hidden, gate_weight, bias)
    return _ext.ops().gate_projection(hidden, gate_weight, bias)


def dispatch_tokens(x: torch.Tensor, logits: torch.Tensor, top_k: int,
                    capacity_factor: float = 1.25, load_balance_weight: float = 0.01,
                    capacity: int | None = None) -> DispatchPlan:
    """:func:`topk_gating_dispatch` with gradients (T >= 1); rows of dropped slots are zero."""
    _ext.require_cuda(x, logits)
    T, E = logits.shape
    C = expert_capacity(T * top_k, E, capacity_factor) if capacity is None else int(capacity)
    outs = _ext.ops().dispatch_tokens(x.half(), logits.float(), int(top_k), C,
                                      float(load_balance_weight),
                                      _ext.error_word(logits.device.index))
    return DispatchPlan(*outs, capacity=C, top_k=int(top_k))


def combine_tokens(expert_output: torch.Tensor, gate_weights: torch.Tensor,
                   plan: DispatchPlan) -> torch.Tensor:
    """:func:`combine` of the plan's rows, ``expert_output`` (T * top_k, d) fp16, with
    gradients.  ``gate_weights`` is the plan's or another (T * top_k,) fp32 tensor; a row that
    no slot keeps gets a zero gradient, a dropped slot's weight too."""
    _ext.require_cuda(expert_output, gate_weights)
    return _ext.ops().combine_tokens(expert_output, gate_weights, plan.slot_pos, plan.offsets,
                                     plan.kept_counts, plan.top_k)

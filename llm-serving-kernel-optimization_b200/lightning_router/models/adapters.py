"""Low-rank adapters of the experts' matrices, one set per (adapter, expert).

``ExpertAdapters`` holds the A and B matrices of ``num_adapters`` adapters for every expert's
gate, up and down projection in the layout of :class:`AdapterBank`, entry ``adapter * E +
expert``.  Attach it to a layer (``layer.adapters = ExpertAdapters(...)``) and pass each
token's adapter number to ``MoELayer.forward(h, adapter_ids=...)``.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from lightning_router.kernels.adapters import AdapterBank

_MATS = ("gate", "up", "down")


class ExpertAdapters(nn.Module):
    def __init__(self, num_adapters: int, num_experts: int, hidden_size: int,
                 intermediate_size: int, rank: int, gated: bool = True):
        super().__init__()
        if rank % 8 or not 8 <= rank <= 128:
            raise ValueError(f"rank must be a multiple of 8 up to 128, got {rank} (pad smaller "
                             "adapters with zeros: load() does)")
        if hidden_size % 8 or intermediate_size % 8:
            raise ValueError("hidden_size and intermediate_size must be multiples of 8")
        if num_adapters < 1 or num_experts < 1:
            raise ValueError("at least one adapter and one expert")
        self.num_adapters, self.num_experts, self.rank = num_adapters, num_experts, rank
        self.hidden_size, self.intermediate_size, self.gated = hidden_size, intermediate_size, gated
        for m in self.mats:
            K, N = (intermediate_size, hidden_size) if m == "down" else (hidden_size,
                                                                         intermediate_size)
            self.register_buffer(f"{m}_a", torch.zeros(num_adapters, num_experts, rank, K,
                                                       dtype=torch.float16))
            self.register_buffer(f"{m}_b", torch.zeros(num_adapters, num_experts, N, rank,
                                                       dtype=torch.float16))
            self.register_buffer(f"{m}_scale", torch.ones(num_adapters, num_experts))

    @property
    def mats(self) -> tuple[str, ...]:
        return _MATS if self.gated else _MATS[1:]

    def check(self, experts) -> None:
        """Refuses the experts (:class:`ExpertGroup`) that these adapters were not made for."""
        mine = (self.num_experts, self.hidden_size, self.intermediate_size, self.gated)
        gated = experts.activation == "swiglu"
        theirs = (experts.num_experts, experts.hidden_size, experts.intermediate_size, gated)
        if mine != theirs:
            raise RuntimeError("adapters for (experts, hidden size, intermediate size, gated) "
                               f"{mine}, the layer has {theirs}")

    @torch.no_grad()
    def load(self, adapter: int, expert: int, mat: str, A: torch.Tensor, B: torch.Tensor,
             scale: float = 1.0) -> None:
        """Adapter matrices A (r, K) and B (N, r), ``r <= rank``, of one expert's projection
        ``mat`` ("gate", "up" or "down"); ``scale`` is usually alpha / r."""
        if mat not in self.mats:
            raise ValueError(f"mat must be one of {self.mats}, got {mat!r}")
        a, b = getattr(self, f"{mat}_a")[adapter, expert], getattr(self, f"{mat}_b")[adapter, expert]
        r = A.shape[0]
        if r > self.rank or A.shape != (r, a.shape[1]) or B.shape != (b.shape[0], r):
            raise ValueError(f"{mat}: A (r <= {self.rank}, {a.shape[1]}) and B ({b.shape[0]}, r) "
                             f"expected, got {tuple(A.shape)} and {tuple(B.shape)}")
        a.zero_()
        b.zero_()
        a[:r].copy_(A)
        b[:, :r].copy_(B)
        getattr(self, f"{mat}_scale")[adapter, expert] = float(scale)

    def bank(self, mat: str) -> AdapterBank:
        a, b = getattr(self, f"{mat}_a"), getattr(self, f"{mat}_b")
        return AdapterBank(a.flatten(0, 1), b.flatten(0, 1),
                           getattr(self, f"{mat}_scale").float().flatten())

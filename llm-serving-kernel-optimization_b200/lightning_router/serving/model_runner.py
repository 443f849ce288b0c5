"""Model runner around the B200 MoE layer, with CUDA-graph replay of fixed shapes.

Same interface as the reference's ``LightningModelRunner``
(``lightning_router/serving/model_runner.py:29-118``): constructed from config
dicts, ``load_model(checkpoint_path)``, ``execute_model(input_ids,
hidden_states) -> output`` per step, and ``enable_profiling`` /
``profile_step``.

The single-GPU layer forward has no host synchronisation (routing, expert GEMMs
and combine are all stream-ordered and size their buffers from static
bounds), so a step of a fixed token count can be captured once as a CUDA graph
and replayed: :meth:`LightningModelRunner.capture` records it, and
``execute_model`` replays it whenever the input has a captured shape (decode
steps do), copying the input into the graph's static buffer.  Other shapes run
eagerly.
"""

from __future__ import annotations

import logging
from pathlib import Path
from typing import Any

import torch

logger = logging.getLogger(__name__)


class _Graph:
    def __init__(self, graph: torch.cuda.CUDAGraph, x: torch.Tensor, out: torch.Tensor,
                 aux: torch.Tensor, ids: torch.Tensor | None = None, adapters=None):
        self.graph, self.x, self.out, self.aux = graph, x, out, aux
        self.ids, self.adapters = ids, adapters   # the adapters that the graph reads
        # the memory it reads, kept for as long as the graph may be replayed
        self.banks = [] if adapters is None else [b.detach() for b in adapters.buffers()]

    def reads(self, adapters) -> bool:
        """Whether these are the adapters captured, in the memory they had then."""
        if adapters is not self.adapters:
            return False
        now = list(adapters.buffers())
        return len(now) == len(self.banks) and all(
            a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.dtype == b.dtype
            and a.stride() == b.stride() for a, b in zip(now, self.banks))


class LightningModelRunner:
    """Runs one MoE layer on one GPU for a serving engine."""

    def __init__(self, model_config: dict[str, Any], moe_config: dict[str, Any],
                 quant_config: dict[str, Any], kernel_config: dict[str, Any],
                 device: torch.device | str = "cuda"):
        self.device = torch.device(device)
        self.model_config = dict(model_config)
        self.moe_config = dict(moe_config)
        self.quant_config = dict(quant_config)
        self.kernel_config = dict(kernel_config)
        self.moe_layer = None
        self._graphs: dict[tuple, _Graph] = {}
        self._pool = None

    # -- model ------------------------------------------------------------
    def load_model(self, checkpoint_path: str | Path | None = None) -> None:
        """Build the MoE layer on the device; load a state dict (packed INT4 buffers
        included) when ``checkpoint_path`` is given, else keep the initial weights."""
        from lightning_router.config import KernelConfig, ModelConfig, MoEConfig, QuantizationConfig
        from lightning_router.models.moe_layer import MoELayer
        layer = MoELayer(ModelConfig(**self.model_config), MoEConfig(**self.moe_config),
                         QuantizationConfig(**self.quant_config),
                         KernelConfig(**self.kernel_config))
        if checkpoint_path is not None:
            state = torch.load(checkpoint_path, map_location="cpu", weights_only=True)
            missing, unexpected = layer.load_state_dict(state, strict=False)
            if unexpected:
                logger.warning("checkpoint entries not used: %s", unexpected)
            logger.info("Loaded checkpoint from %s", checkpoint_path)
        layer = layer.to(self.device)
        layer.gate.gate_proj.half()  # the gate GEMM reads fp16 weights (bias stays fp32)
        self.moe_layer = layer.eval()
        self._graphs.clear()

    def set_adapters(self, adapters) -> None:
        """Serve these low-rank adapters (:class:`ExpertAdapters`; ``None``: no more).
        Graphs captured with the former ones are dropped."""
        layer = self._layer()
        layer.adapters = None if adapters is None else adapters.to(self.device)
        self._graphs = {k: g for k, g in self._graphs.items() if g.ids is None}

    # -- execution --------------------------------------------------------
    @torch.inference_mode()
    def capture(self, num_tokens: int, warmup: int = 2, adapters: bool = False) -> None:
        """Record one forward of ``num_tokens`` tokens as a CUDA graph (after
        ``warmup`` eager runs, which build the weight tables and size the caches).
        With ``adapters`` the graph takes adapter numbers too."""
        layer = self._layer()
        d = layer.hidden_size
        key = (num_tokens, d, True) if adapters else (num_tokens, d)
        ids = torch.full((num_tokens,), -1, dtype=torch.int32, device=self.device) \
            if adapters else None
        kw = {} if ids is None else {"adapter_ids": ids}   # a layer may know of none
        x = torch.zeros(num_tokens, d, dtype=torch.float16, device=self.device)
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            for _ in range(max(1, warmup)):
                layer(x, **kw)
        torch.cuda.current_stream(self.device).wait_stream(side)
        torch.cuda.synchronize(self.device)
        if self._pool is None:
            self._pool = torch.cuda.graph_pool_handle()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=self._pool):
            out, aux = layer(x, **kw)
        self._graphs[key] = _Graph(g, x, out, aux, ids, layer.adapters if adapters else None)

    @torch.inference_mode()
    def execute_model(self, input_ids: torch.Tensor | None,
                      hidden_states: torch.Tensor,
                      adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
        """One step through the MoE layer: (..., hidden) -> (..., hidden).
        ``input_ids`` is accepted for interface compatibility and not used;
        ``adapter_ids`` gives each token its adapter (:meth:`set_adapters`), -1 for none."""
        layer = self._layer()
        shape = hidden_states.shape
        h = hidden_states.reshape(-1, shape[-1])
        key = (h.shape[0], h.shape[1])
        gr = self._graphs.get(key if adapter_ids is None else (*key, True))
        if gr is not None and gr.ids is not None and not gr.reads(layer.adapters):
            gr = None   # captured with adapters that the layer no longer has, or has elsewhere
        if gr is None:
            out, _ = layer(h) if adapter_ids is None else layer(h, adapter_ids=adapter_ids)
            return out.view(shape).to(hidden_states.dtype)
        if adapter_ids is not None:
            from lightning_router.kernels.adapters import adapter_index
            if adapter_ids.numel() != h.shape[0]:
                raise ValueError(f"adapter_ids has {adapter_ids.numel()} entries for "
                                 f"{h.shape[0]} tokens")
            gr.ids.copy_(adapter_index(adapter_ids))
        gr.x.copy_(h)
        gr.graph.replay()
        return gr.out.clone().view(shape).to(hidden_states.dtype)

    # -- profiling --------------------------------------------------------
    def enable_profiling(self) -> None:
        self._prof_start = torch.cuda.Event(enable_timing=True)
        self._prof_end = torch.cuda.Event(enable_timing=True)

    def profile_step(self, hidden_states: torch.Tensor) -> dict[str, float]:
        """One step with CUDA-event timing of the whole layer (ms)."""
        if not hasattr(self, "_prof_start"):
            self.enable_profiling()
        self._prof_start.record()
        self.execute_model(None, hidden_states)
        self._prof_end.record()
        torch.cuda.synchronize(self.device)
        return {"moe_layer_ms": self._prof_start.elapsed_time(self._prof_end)}

    def _layer(self):
        if self.moe_layer is None:
            raise RuntimeError("load_model() has not been called")
        return self.moe_layer

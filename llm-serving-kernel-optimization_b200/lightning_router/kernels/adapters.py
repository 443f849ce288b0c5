"""Low-rank adapters of many requests at once beside a shared projection.

One batch mixes the rows of many requests; row t carries an adapter number (or -1).  The
projection runs once for all rows (:func:`quantized_matmul` or any other), and

* :func:`adapter_add` adds ``scale_a (x_t A_a^T) B_a^T`` to its rows;
* :func:`adapter_swiglu` does so beside a SwiGLU expert's gate and up projections and takes
  ``silu(gate) * up``;
* :func:`adapter_rows` numbers the rows of an expert dispatch for a bank that holds one
  adapter per (request's adapter, expert);
* :func:`quantized_matmul_adapters` is the INT4 projection with its adapters.

Rows come in any order; neighbours with the same adapter share its weights' reads, so a
prompt's rows belong next to each other.  ``x A^T`` is kept in fp32, sums are fp32, the result
is rounded to fp16 once.  A row's result depends on its own adapter only, whatever the others
hold.  Serving operators: no backward (inputs that require a gradient are refused).
"""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from lightning_router import _ext
from lightning_router.kernels.quantized_matmul import quantized_matmul


class AdapterBank(NamedTuple):
    """``n`` adapters of one projection K -> N; K, N and the rank (at most 128) multiples of 8.

    Contiguous fp16 ``a`` (n, rank, K) and ``b`` (n, N, rank), the layout of the usual A and B
    matrices, and fp32 ``scale`` (n,), usually alpha / rank (``None``: 1)."""
    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor | None = None


def pack_adapters(pairs: Sequence[tuple[torch.Tensor, torch.Tensor]],
                  scales: Sequence[float] | None = None) -> AdapterBank:
    """A bank from (A (rank_i, K), B (N, rank_i)) pairs whose ranks may differ: ranks are
    padded with zeros to the largest one's next multiple of 8."""
    if not pairs:
        raise ValueError("pack_adapters: no adapters")
    if scales is not None and len(scales) != len(pairs):
        raise ValueError(f"pack_adapters: {len(pairs)} adapters and {len(scales)} scales")
    K, N = pairs[0][0].shape[1], pairs[0][1].shape[0]
    for A, B in pairs:
        if A.dim() != 2 or B.dim() != 2 or A.shape[1] != K or B.shape != (N, A.shape[0]):
            raise ValueError(f"pack_adapters: A (rank, {K}) and B ({N}, rank) expected, got "
                             f"{tuple(A.shape)} and {tuple(B.shape)}")
    rank = max(A.shape[0] for A, _ in pairs)
    rank = max(8, -(-rank // 8) * 8)
    dev = pairs[0][0].device
    a = torch.zeros(len(pairs), rank, K, dtype=torch.float16, device=dev)
    b = torch.zeros(len(pairs), N, rank, dtype=torch.float16, device=dev)
    for i, (A, B) in enumerate(pairs):
        a[i, :A.shape[0]] = A
        b[i, :, :A.shape[0]] = B
    scale = None if scales is None else torch.tensor([float(v) for v in scales],
                                                     dtype=torch.float32, device=dev)
    return AdapterBank(a, b, scale)


def _no_grad(name: str, *tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad() or detach "
                           "its inputs")


def adapter_index(index: torch.Tensor) -> torch.Tensor:
    """Adapter numbers of any integer type as contiguous int32."""
    if index.dtype == torch.int32 and index.dim() == 1 and index.is_contiguous():
        return index
    if index.dtype.is_floating_point or index.dtype.is_complex or index.dtype == torch.bool:
        raise ValueError(f"adapter numbers must be integers, got {index.dtype}")
    if index.dtype in (torch.int64, torch.uint32, torch.uint64):
        wide = index.to(torch.int64)
        if index.dtype == torch.uint64:     # from 2^63 on: negative now, and not "none"
            wide = torch.where(wide < 0, 2**31 - 1, wide)
        index = wide.clamp(-2, 2**31 - 1)   # out of range stays out of range
    return index.reshape(-1).to(torch.int32).contiguous()


def adapter_add(base: torch.Tensor, x: torch.Tensor, bank: AdapterBank, index: torch.Tensor,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``base + scale (x A^T) B^T`` with each row's adapter ``index`` (R,) integers, -1: none.

    ``x`` (R, K) and ``base`` (R, N) fp16.  ``out`` (contiguous) may be ``base`` itself; rows
    without an adapter are then left as they are.  Writing to it counts as an in-place change:
    a backward pass that needs its former values raises.  A number outside [-1, n) is taken as -1 and
    flagged (:func:`lightning_router._ext.check_device_errors`)."""
    _ext.require_cuda(base, x, index, *bank)
    _no_grad("adapter_add", base, x, *bank, out)
    args = (x, adapter_index(index), bank.a, bank.b, bank.scale, base)
    err = _ext.error_word(x.device.index)
    if out is None:
        return _ext.ops().adapter_add(*args, err)
    _ext.ops().adapter_add_out(*args, out, err)
    return out


def adapter_swiglu(gate: torch.Tensor, up: torch.Tensor, x: torch.Tensor, gate_bank: AdapterBank,
                   up_bank: AdapterBank, index: torch.Tensor,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(gate + delta_gate) * (up + delta_up)`` with each row's adapters; see
    :func:`adapter_add`.  The banks have the same n, rank and sizes."""
    _ext.require_cuda(gate, up, x, index, *gate_bank, *up_bank)
    _no_grad("adapter_swiglu", gate, up, x, *gate_bank, *up_bank, out)
    args = (x, adapter_index(index), *gate_bank, *up_bank, gate, up)
    err = _ext.error_word(x.device.index)
    if out is None:
        return _ext.ops().adapter_swiglu(*args, err)
    _ext.ops().adapter_swiglu_out(*args, out, err)
    return out


def adapter_rows(adapter_ids: torch.Tensor, plan, num_adapters: int) -> torch.Tensor:
    """Per row of a dispatch ``plan`` the entry ``adapter * E + expert`` of a bank with one
    adapter per expert, from the tokens' ``adapter_ids`` (T,) in [-1, num_adapters).  Dropped
    rows and tokens without an adapter get -1."""
    _ext.require_cuda(adapter_ids, plan.source_indices)
    return _ext.ops().adapter_rows(adapter_index(adapter_ids), plan.source_indices, plan.offsets,
                                   plan.kept_counts, int(num_adapters),
                                   _ext.error_word(adapter_ids.device.index))


def quantized_matmul_adapters(A: torch.Tensor, B_packed: torch.Tensor, scales: torch.Tensor,
                              zeros: torch.Tensor, N: int, bank: AdapterBank,
                              index: torch.Tensor, group_size: int = 128) -> torch.Tensor:
    """:func:`quantized_matmul` with the rows' adapters added to its result in place."""
    base = quantized_matmul(A, B_packed, scales, zeros, N, group_size)
    return adapter_add(base, A, bank, index, out=base)

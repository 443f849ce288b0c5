"""Adapter numbers of every integer type: what is out of range stays out of range."""

from __future__ import annotations

import pytest
import torch

from lightning_router.kernels.adapters import adapter_index


@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.int32, torch.int64])
def test_signed(dtype):
    t = torch.tensor([-1, 0, 5, -2, 127], dtype=dtype)
    assert adapter_index(t).tolist() == [-1, 0, 5, -2, 127] and adapter_index(t).dtype == torch.int32


@pytest.mark.parametrize("dtype,top", [(torch.uint8, 255), (torch.uint16, 65535),
                                       (torch.uint32, 2**32 - 1), (torch.uint64, 2**64 - 1)])
def test_unsigned(dtype, top):
    got = adapter_index(torch.tensor([0, 7, top], dtype=dtype)).tolist()
    assert got[:2] == [0, 7] and got[2] == min(top, 2**31 - 1)


def test_wide():
    t = torch.tensor([2**31, -2**31 - 5, 2**62, -2**63])
    assert adapter_index(t).tolist() == [2**31 - 1, -2, 2**31 - 1, -2]
    u = torch.tensor([2**63, 2**63 + 3, 2**32], dtype=torch.uint64)
    assert adapter_index(u).tolist() == [2**31 - 1] * 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bool, torch.complex64])
def test_refused(dtype):
    with pytest.raises(ValueError, match="integers"):
        adapter_index(torch.zeros(3, dtype=dtype))

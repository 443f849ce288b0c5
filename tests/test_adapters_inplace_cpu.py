"""The adapters' ops name the tensor that they write to."""

from __future__ import annotations

import pytest

from lightning_router import _ext


@pytest.mark.parametrize("op", ["adapter_add", "adapter_swiglu"])
def test_schemas(op):
    ops = _ext.ops()
    plain = getattr(ops, op).default._schema
    assert not any(a.name == "out" for a in plain.arguments)
    assert not any(a.alias_info for a in plain.arguments) and len(plain.returns) == 1
    out = getattr(ops, op + "_out").default._schema
    written = [a.name for a in out.arguments if a.alias_info and a.alias_info.is_write]
    assert written == ["out"] and not out.returns and out.is_mutable

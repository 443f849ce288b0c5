"""Waits that a whole warp makes end with one verdict for all of its lanes.

A bounded wait may time out, or see another warp's abort, in some lanes and complete in others.
Lanes that then leave a loop while the rest run ``mma.sync`` or a full-mask ``__syncwarp`` hang
or compute nonsense, so the whole-warp waits vote.  No GPU can show that without being hung:
the source is checked.
"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "llm-serving-kernel-optimization_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def _body(code, head):
    """The text of the function whose definition starts with ``head``."""
    at = code.index("{", code.index(head))
    depth = 0
    for i in range(at, len(code)):
        depth += {"{": 1, "}": -1}.get(code[i], 0)
        if depth == 0:
            return code[at:i + 1]
    raise AssertionError(head)


def test_the_warp_wait_votes():
    body = _body(_code("lr_common.cuh"), "bool mbar_wait_warp(")
    assert re.search(r"__all_sync\(0xffffffffu,\s*mbar_wait_bounded\(", body)


@pytest.mark.parametrize("name", ["lr_lowrank.cuh", "lr_adapters.cu", "lr_router_grad.cu"])
def test_whole_warp_waits_use_it(name):
    code = _code(name)
    assert "mbar_wait_bounded" not in code and "mbar_try_wait" not in code
    if name == "lr_lowrank.cuh":
        assert code.count("mbar_wait_warp(") == 2     # the producer's and the consumers'


def test_cluster_barrier_gathers_the_warp():
    body = _body(_code("lr_lowrank.cuh"), "void cluster_sync()")
    assert body.index("__syncwarp()") < body.index("barrier.cluster.arrive")


@pytest.mark.parametrize("name,loop", [("lr_w4a16_gemm.cu", "for (; kb < KB; kb += DGROUPS)"),
                                       ("lr_w4a16_skinny.cu", "for (int kb = 0; kb < KB; ++kb) {")])
def test_gemm_lanes_stay_in_step(name, loop):
    """The loops of whole warps in the GEMMs take no vote at each wait: a lane whose wait ran out
    goes on to the end with the others, so none leaves ahead of mma.sync or __syncwarp, and its
    warp's lane 0 arrives only while its own waits held."""
    code = _code(name)
    body = _body(code, loop)
    assert "wait_any(" in body and "__syncwarp" in body
    assert "break" not in body and "return" not in body
    assert len(re.findall(r"if \(lane == 0\)", body)) == 0
    assert "if (lane == 0 && ok)" in body

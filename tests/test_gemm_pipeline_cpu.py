"""The W4A16 GEMM's rings against every order in which copies may land.

An mbarrier wait looks at one bit, the parity of the phase.  A waiter that is a whole phase ahead
of the barrier reads "complete".  The packed-weight stages are read by warp groups that take
alternate k-steps, so a stage passes from group to group wherever the number of groups does not
divide the number of stages, and copies may land in any order.  The model runs producer, groups
and MMA in random interleavings with random landings and checks that a group only ever reads the
words of its own k-step and that no barrier is armed twice in a phase.  The tile shapes, the
number of "words loaded" barriers and the order of the group's two waits are taken from the source.
"""

from __future__ import annotations

import math
import random
import re
from pathlib import Path

import pytest

SRC = (Path(__file__).resolve().parents[1] / "llm-serving-kernel-optimization_b200" / "csrc"
       / "lr_w4a16_gemm.cu").read_text()
CODE = re.sub(r"//[^\n]*", "", SRC)

SHAPES = {m[0]: tuple(int(v) for v in m[1].split(","))[3:] for m in
          re.findall(r"using (Shape\w+) = GemmShape<([\d, ]+)>", CODE)}


def waits_in_source() -> tuple[str, str]:
    """The dequant loop's barriers in the order in which it waits for them."""
    loop = CODE[CODE.index("for (; kb < KB; kb += DGROUPS)"):]
    loop = loop[:loop.index("__syncwarp")]
    names = re.findall(r"wait_any\(&(\w+)\[", loop)
    assert sorted(names) == ["empty", "wfull"], names
    return tuple(names)


def barriers_in_source(stages: int, groups: int) -> int:
    """"Words loaded" barriers of a shape: one per stage, or one per stage and group."""
    uses = re.findall(r"wfull\[([^\]]+)\]", CODE[CODE.index("auto decode = "):])
    if set(uses) == {"it % S::WBARS", "i % S::WBARS"}:
        assert "WBARS = least_common_multiple(STAGES, DGROUPS)" in CODE
        return math.lcm(stages, groups)
    assert set(uses) == {"s", "i % STAGES"}, uses
    return stages


class Barrier:
    """Phases completed so far; ``wait(parity)`` as the hardware answers it."""

    def __init__(self, count):
        self.count, self.done, self.pending, self.tx = count, 0, count, 0

    def wait(self, parity):
        return (self.done & 1) != parity

    def arrive(self, tx=0):
        assert self.pending > 0, "armed twice in one phase"
        self.pending -= 1
        self.tx += tx
        self._complete()

    def landed(self):
        self.tx -= 1
        self._complete()

    def _complete(self):
        if self.pending == 0 and self.tx == 0:
            self.done += 1
            self.pending = self.count


def run(stages, dstages, groups, wbars, order, steps, seed):
    """One random schedule; raises AssertionError on a wrong read or a double arrival."""
    rnd = random.Random(seed)
    wfull = [Barrier(1) for _ in range(wbars)]
    wempty = [Barrier(1) for _ in range(stages)]
    empty = [Barrier(1) for _ in range(stages)]
    dfull = [Barrier(1) for _ in range(dstages)]
    words = [None] * stages            # the k-step whose words a stage holds
    flying = []                        # copies on their way
    slow = [rnd.random() for _ in range(stages)]
    land, pick = rnd.choice([0.02, 0.1, 0.4]), rnd.choice([1, 2, stages])

    def producer():
        for it in range(steps):
            s = it % stages
            while not wempty[s].wait((it // stages & 1) ^ 1):
                yield
            wfull[it % wbars].arrive(tx=1)
            flying.append(it)
            yield

    def group(g):
        for it in range(g, steps, groups):
            s, q, prev = it % stages, it % dstages, it - dstages
            for name in order:
                if name == "wfull":
                    while not wfull[it % wbars].wait(it // wbars & 1):
                        yield
                elif prev >= 0:
                    while not empty[prev % stages].wait(prev // stages & 1):
                        yield
                yield
            assert words[s] == it, f"read the words of k-step {words[s]} for {it}"
            wempty[s].arrive()
            yield
            dfull[q].arrive()
            yield

    def mma():
        for it in range(steps):
            while not dfull[it % dstages].wait(it // dstages & 1):
                yield
            yield
            empty[it % stages].arrive()

    actors = [producer(), mma()] + [group(g) for g in range(groups)]
    weights = [rnd.choice([1, 4, 16]) for _ in actors]
    idle = 0
    while actors:
        # copies land in any order, some stages' later than others'
        if flying and rnd.random() < land:
            it = min(rnd.sample(flying, min(pick, len(flying))), key=lambda i: slow[i % stages])
            flying.remove(it)
            words[it % stages] = it
            wfull[it % wbars].landed()
            idle = 0
            continue
        i = rnd.choices(range(len(actors)), weights)[0]
        try:
            next(actors[i])
        except StopIteration:
            del actors[i], weights[i]
            idle = 0
        idle += 1
        assert idle < 100000, "stuck"


def test_shapes_were_found():
    assert SHAPES["ShapeR256W"] == (3, 3, 2) and len(SHAPES) >= 5
    assert all(d <= s for s, d, _ in SHAPES.values())


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_every_group_reads_its_own_words(name):
    stages, dstages, groups = SHAPES[name]
    for seed in range(300):
        run(stages, dstages, groups, barriers_in_source(stages, groups), waits_in_source(), 80, seed)


def test_the_model_finds_one_barrier_per_stage():
    """Where stages pass between groups, a wait for the words ahead of the one for the buffer
    then reads other words."""
    found = set()
    for name, (stages, dstages, groups) in SHAPES.items():
        for seed in range(300):
            try:
                run(stages, dstages, groups, stages, ("wfull", "empty"), 40, seed)
            except AssertionError:
                found.add(name)
                break
    assert found == {n for n, (s, _, g) in SHAPES.items() if s % g}

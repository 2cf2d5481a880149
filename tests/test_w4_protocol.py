"""The barriers of the 4-bit tensor-core kernel, simulated.

Its unpacking groups take every G-th block, so a group does not see every
phase of a barrier it waits on. A parity wait cannot tell a phase from the one
two before it: the simulation runs the producers, the groups and the MMA issuer
in random orders and checks that no wait is let through in a phase other than
the one it is for, and that the work ends, for every number of groups that the
kernel's rule allows (the rule is read from the source).
"""

from __future__ import annotations

import pathlib
import random
import re

import pytest

SRC = pathlib.Path(__file__).resolve().parents[1] / "flash-head_b200" / "csrc" / "fh_w4_tc.cuh"


def rule():
    text = SRC.read_text()
    most = int(re.search(r"kW4tGroups = (\d+)", text).group(1))
    cond = re.search(r"while \(g > 0 && \((.*)\)\) --g;", text).group(1).replace("||", "or")

    def groups(stages, packed):
        g = most
        while g > 0 and eval(cond, {}, {"g": g, "stages": stages, "packed": packed}):
            g -= 1
        return g
    return groups


class Ambiguous(Exception):
    pass


class Bar:
    """An mbarrier: `phase` phases are complete."""

    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left = self.count
            self.phase += 1

    def ok(self, k):
        """A parity wait for phase k (k < 0: passes at once)."""
        if k < 0:
            if self.phase > 1:
                raise Ambiguous
            return True
        passes = (self.phase & 1) != (k & 1)
        if passes != (self.phase > k):
            raise Ambiguous
        return passes


def simulate(blocks, stages, packed, groups, seed):
    rnd = random.Random(seed)
    full = [Bar(2) for _ in range(stages)]
    empty = [Bar(1) for _ in range(stages)]
    pfull = [Bar(1) for _ in range(packed)]
    pempty = [Bar(1) for _ in range(packed)]
    copies, mmas = [], []

    def packed_producer():
        for n in range(blocks):
            while not pempty[n % packed].ok(n // packed - 1):
                yield
            copies.append(pfull[n % packed])
            yield

    def hidden_producer():
        for n in range(blocks):
            while not empty[n % stages].ok(n // stages - 1):
                yield
            copies.append(full[n % stages])
            yield

    def unpack(g):
        for n in range(g, blocks, groups):
            while not pfull[n % packed].ok(n // packed):
                yield
            yield
            pempty[n % packed].arrive()
            while not empty[n % stages].ok(n // stages - 1):
                yield
            yield
            full[n % stages].arrive()
            yield

    def issue():
        for n in range(blocks):
            while not full[n % stages].ok(n // stages):
                yield
            mmas.append(empty[n % stages])
            yield

    agents = [packed_producer(), hidden_producer(), issue()] + [unpack(g) for g in range(groups)]
    speed = [rnd.choice([0.02, 0.2, 1, 3]) for _ in agents]
    for _ in range(200000):
        if not agents:
            return
        r = rnd.random()
        if mmas and r < 0.15:  # in order
            mmas.pop(0).arrive()
        elif copies and r < 0.4:  # in any order
            copies.pop(rnd.randrange(len(copies))).arrive()
        else:
            i = rnd.choices(range(len(agents)), speed)[0]
            try:
                next(agents[i])
            except StopIteration:
                agents.pop(i)
                speed.pop(i)
    raise AssertionError("stuck")


@pytest.mark.parametrize("stages", [2, 3, 4])
@pytest.mark.parametrize("packed", [3, 5, 6, 8, 12])
def test_allowed_groups_never_pass_early(stages, packed):
    groups = rule()(stages, packed)
    assert groups <= stages
    for seed in range(12 if groups else 0):
        simulate(40, stages, packed, groups, seed)


def test_the_simulation_finds_too_many_groups():
    """Three groups on two stages: a group may skip a phase of a stage."""
    with pytest.raises((Ambiguous, AssertionError)):
        for seed in range(200):
            simulate(40, 2, 4, 3, seed)

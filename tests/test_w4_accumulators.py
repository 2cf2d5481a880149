"""The whole protocol of the 4-bit tensor-core kernel with an accumulator per
block, simulated: packed blocks, unpacking groups, two issuing warps with
accumulators of their own, summing warps and the slots in which scales are
handed on. The rule of the other kernel's unpacking groups goes through the
simulation of one issuing warp.

Random orders; checked are that no parity wait passes early, that scales and
accumulators hold what their reader expects, and that the work ends.
"""

from __future__ import annotations

import pathlib
import random
import re

import pytest

import test_w4_protocol as protocol
from test_w4_protocol import Ambiguous, Bar, rule

re_search = re.search
SRC = pathlib.Path(__file__).resolve().parents[1] / "flash-head_b200" / "csrc" / "fh_w4_tc.cuh"


def constant(name):
    return int(re.search(rf"constexpr int {name} = (\d+)", SRC.read_text()).group(1))


STAGES, SLOTS, ACC = (constant(n) for n in ("kW4tStages", "kW4tScaleSlots", "kW4tMaxAcc"))


def simulate(blocks, packed, groups, n_acc, sums, seed, slots=SLOTS, stages=STAGES):
    rnd = random.Random(seed)
    hfull = [Bar(1) for _ in range(stages)]
    full = [Bar(1) for _ in range(stages)]
    empty = [Bar(1) for _ in range(stages)]
    pfull = [Bar(1) for _ in range(packed)]
    pempty = [Bar(1) for _ in range(packed)]
    afull = [[Bar(1) for _ in range(n_acc)] for _ in range(2)]
    aempty = [[Bar(sums) for _ in range(n_acc)] for _ in range(2)]
    scales, acc, a_tile, words = {}, {}, {}, {}
    copies, mmas = [], []

    def loader(bar_full, bar_empty, ring, land):
        for n in range(blocks):
            while not bar_empty[n % ring].ok(n // ring - 1):
                yield
            copies.append((bar_full[n % ring], land, n))
            yield

    def unpack(g):
        for n in range(g, blocks, groups):
            while not pfull[n % packed].ok(n // packed):
                yield
            assert words[n % packed] == n
            pempty[n % packed].arrive()
            while not empty[n % stages].ok(n // stages - 1):
                yield
            scales[n % slots] = n
            yield
            a_tile[n % stages] = n
            full[n % stages].arrive()
            yield

    def issue(mine):
        use = 0
        for n in range(mine, blocks, 2):
            st, k = n % stages, n // stages
            for bars in (hfull, full):
                while not bars[st].ok(k):
                    yield
            while not aempty[mine][use % n_acc].ok(use // n_acc - 1):
                yield
            mmas.append(("mma", mine, use % n_acc, n))
            mmas.append(("commit", afull[mine][use % n_acc]))
            mmas.append(("commit", empty[st]))
            use += 1
            yield

    def add():
        use = [0, 0]
        for n in range(blocks):
            odd = n % 2
            slot, k = use[odd] % n_acc, use[odd] // n_acc
            while not afull[odd][slot].ok(k):
                yield
            assert acc[odd, slot] == n and scales[n % slots] == n
            yield
            assert acc[odd, slot] == n
            aempty[odd][slot].arrive()
            use[odd] += 1
            yield

    agents = [loader(pfull, pempty, packed, lambda n: words.__setitem__(n % packed, n)),
              loader(hfull, empty, stages, lambda n: None), issue(0), issue(1)]
    agents += [unpack(g) for g in range(groups)] + [add() for _ in range(sums)]
    speed = [rnd.choice([0.02, 0.2, 1, 3]) for _ in agents]
    for _ in range(400000):
        if not agents:
            return
        r = rnd.random()
        if mmas and r < 0.25:  # in the order of their issue
            op = mmas.pop(0)
            if op[0] == "mma":
                _, mine, slot, n = op
                assert a_tile[n % stages] == n
                acc[mine, slot] = n
            else:
                op[1].arrive()
        elif copies and r < 0.5:
            bar, land, n = copies.pop(rnd.randrange(len(copies)))
            land(n)
            bar.arrive()
        else:
            i = rnd.choices(range(len(agents)), speed)[0]
            try:
                next(agents[i])
            except StopIteration:
                agents.pop(i)
                speed.pop(i)
    raise AssertionError("stuck")


@pytest.mark.parametrize("packed,most,n_acc,sums", [
    (12, 4, ACC, 1), (12, 4, ACC, 2), (8, 2, 1, 3), (8, 2, 1, 4)])
def test_the_launched_shapes(packed, most, n_acc, sums):
    groups = min(rule()(STAGES, packed), most)
    assert groups == most
    for seed in range(20):
        simulate(40, packed, groups, n_acc, sums, seed)


@pytest.mark.parametrize("blocks", [1, 2, 3])
def test_short_work(blocks):
    for seed in range(20):
        simulate(blocks, 12, 4, ACC, 2, seed)


def test_the_simulation_finds_too_few_scale_slots():
    with pytest.raises(AssertionError):
        for seed in range(200):
            simulate(40, 12, 4, ACC, 1, seed, slots=6)


def test_the_simulation_finds_groups_that_skip_phases():
    with pytest.raises((Ambiguous, AssertionError, KeyError)):
        for seed in range(200):
            simulate(40, 8, 3, ACC, 1, seed)


@pytest.mark.parametrize("stages", [2, 3])
@pytest.mark.parametrize("packed", [4, 5, 6, 8, 9, 12])
def test_the_other_kernels_groups(stages, packed, monkeypatch):
    monkeypatch.setattr(protocol, "SRC", SRC.with_name("fh_w4_split.cuh"))
    monkeypatch.setattr(protocol.re, "search", lambda pat, text: re_search(
        pat.replace("kW4tGroups", "kW4sGroups"), text))
    groups = rule()(stages, packed)
    assert 1 <= groups <= stages
    for seed in range(12):
        protocol.simulate(40, stages, packed, groups, seed)

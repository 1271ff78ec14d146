"""The counting wait of the 4-bit products in tiles (``mx4_tiles_kernel``), under the check of ``test_load_order``.

A step waits until no more loads are on their way than the rings asked for behind the step's own two stages.  Loads of scales, which go to registers, are not in that count: the compiler
moves them among the others as it likes, and a count that took some of them for granted would let a step read a stage that is not there.  So: the rings' loads stand in their order, in front
of the loop and in it, and the wait in front of the barrier is their number alone."""
from __future__ import annotations

import re

import pytest

from test_load_order import events, kernels, parts, places, waits_at_barriers

SHAPE = r"MtShapeILb(\d)E" + r"Li(\d+)E" * 7


def shape_of(name):
    return [int(x) for x in re.search(SHAPE, name).groups()]


def check(rows, four, ft, tt, wf, wt, sf, st, planes):
    waves = wf * wt
    f = 32 * ft * wf * (8 if four else 2) // 64 // waves              # loads of a wave and stage, of features and of tokens
    t = planes * 32 * tt * wt * 8 // 64 // waves
    front, loop, behind = parts(rows)
    rings = [e for e in loop if e[0] == "lds"]
    assert rings == [rings[0]] * t + [rings[-1]] * f and rings[0] != rings[-1]
    # (the registers that hold the buffers may be others in front of the loop)
    before = [e for e in front if e[0] == "lds"]
    features = before[-1]
    tokens, = {e for e in before if e != features}
    assert before == [features] * f * (sf - st) + ([tokens] * t + [features] * f) * (st - 1)
    assert waits_at_barriers(loop) == [(f if sf > st else 0) + (st - 2) * (f + t)]
    # the barrier is in front of the step's loads, which go where the step before was read from
    kinds = [k for k, _ in loop]
    assert kinds.count("barrier") == 1 and kinds.index("barrier") < kinds.index("lds")
    assert "lds" not in [k for k, _ in behind] and waits_at_barriers(behind) == [0]


def test_rings_of_four_bits(tmp_path):
    found = {n: r for n, r in kernels("mx4_tiles", tmp_path).items() if "mx4_tiles_kernel" in n}
    assert len(found) == 48
    for name, rows in found.items():
        check(rows, *shape_of(name))


@pytest.mark.parametrize("part", ["Lb0ELi2ELi1ELi2ELi2ELi4ELi4ELi1E", "Lb0ELi2ELi4ELi4ELi2ELi4ELi3ELi1E", "Lb1ELi2ELi2ELi2ELi2ELi4ELi4ELi1E"])
def test_planted_mistakes_are_found(part, tmp_path):
    """In a copy of the listing: a count that is one too high, a load of tokens behind one of features, a load that is gone, and a load in front of the barrier."""
    name, rows = next((n, r) for n, r in kernels("mx4_tiles", tmp_path).items() if part in n)
    check(rows, *shape_of(name))
    lds, (barrier,) = places(rows, "lds"), places(rows, "barrier")
    wait = max(i for i in places(rows, "wait") if i < barrier)
    first = next(i for i, _ in enumerate(rows) if events(rows[i:i + 1]) and events(rows[i:i + 1])[0][0] == "lds")

    def swapped(i, j):
        r = list(rows)
        r[i], r[j] = r[j], r[i]
        return r

    def instead(i, row):
        return rows[:i] + [row] + rows[i + 1:]
    for bad in (instead(wait, (rows[wait][0], re.sub(r"vmcnt\((\d+)\)", lambda m: f"vmcnt({int(m.group(1)) + 1})", rows[wait][1]), None)), swapped(lds[0], lds[-1]),
                instead(lds[0], ("s_nop", "0", None)), instead(first, ("s_nop", "0", None)), swapped(barrier, lds[0])):
        with pytest.raises((AssertionError, ValueError)):
            check(bad, *shape_of(name))

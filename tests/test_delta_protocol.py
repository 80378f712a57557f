"""The barriers between the roles of the gated delta rule's recurrences, on the CPU.

A wait by parity passes when the barrier's present phase has the other parity: a warp that comes to its wait for phase i
after phase i + 1 has completed as well waits for a phase that needs the warp itself.  So no barrier may complete phase
i + 1 before all who wait for phase i have seen it.  Waits and arrivals only ever enable others, so the furthest that all
other warps come while one stands in front of a wait is found by running them until nothing moves.
"""
import os
import re

import pytest

import aussm_b200

SOURCE = os.path.join(os.path.dirname(aussm_b200.__file__), "csrc", "delta_scan.cu")
CHUNKS = 6


def barriers():
    """Names of the kernel's barriers and how many phases' worth of each there are."""
    text = open(SOURCE).read()
    found = {}
    for line in re.findall(r"__shared__ uint64_t ([^;]+);", text):
        for name, size in re.findall(r"(\w+)(?:\[(\d+)\])?", line):
            found[name] = int(size or 1)
    return found


def programs(backward, full):
    """The roles' waits ("w", barrier, chunk) and arrivals ("a", ...), chunk after chunk.  Two warps stand for the eight that
    own the state; row_s, row_n, v_loaded and v_read only join the threads of one role."""
    main, into, out, copy, issue = [], [], [], [], []
    for i in range(CHUNKS):
        w, a = (lambda p, b, c=i: p.append(("w", b, c))), (lambda p, b, c=i: p.append(("a", b, c)))
        a(main, "s_ready"); w(main, "v_done"); w(main, "v_ready")
        if full and i: w(main, "x_free", i - 1)
        a(main, "n_ready")
        if backward: w(main, "a_done"); a(main, "y_free")
        w(main, "d_done")

        if i: w(into, "a_done" if backward else "v_done", i - 1)
        a(into, "v_ready")

        if full: w(out, "n_ready"); w(out, "o_done"); a(out, "o_free"); a(out, "x_free")

        if i: w(copy, "empty_a", i - 1)
        a(copy, "full_a")
        if i >= 2: w(copy, "empty_b", i - 2)
        if i >= 2 and full: w(copy, "empty_e", i - 2)
        a(copy, "full_b")
        if full: a(copy, "full_e")
        if full or backward:
            if i: w(copy, "empty_c", i - 1)
            a(copy, "full_c")

        w(issue, "full_a"); w(issue, "v_ready")
        if full and i: w(issue, "o_free", i - 1)
        w(issue, "s_ready"); a(issue, "v_done"); a(issue, "empty_a")
        if backward:
            w(issue, "full_c")
            if full and i: w(issue, "x_free", i - 1)
            a(issue, "a_done"); a(issue, "empty_c"); w(issue, "y_free")
        w(issue, "full_b")
        if full:
            w(issue, "full_e")
            if not backward: w(issue, "full_c")
            if i: w(issue, "x_free", i - 1)
        w(issue, "n_ready"); a(issue, "d_done"); a(issue, "empty_b")
        if full:
            if not backward: a(issue, "empty_c")
            a(issue, "o_done"); a(issue, "empty_e")
    return dict(main0=main, main1=list(main), into=into, out=out, copy=copy, issue=issue)


def furthest(progs, frozen=None, at=None):
    """Phases completed per barrier when `frozen` stays in front of its step `at` and all others run as far as they can."""
    count = {n: 0 for n in progs}
    needed = {}
    for n, p in progs.items():
        for kind, b, c in p:
            if kind == "a":
                needed.setdefault((b, c), set()).add(n)
    arrived = {}
    moved = True
    while moved:
        moved = False
        for n, p in progs.items():
            while count[n] < len(p) and not (n == frozen and count[n] == at):
                kind, b, c = p[count[n]]
                if kind == "w" and arrived.get((b, c), set()) != needed[(b, c)]:
                    break
                if kind == "a":
                    arrived.setdefault((b, c), set()).add(n)
                count[n] += 1
                moved = True
    done = {}
    for (b, c), who in needed.items():
        if arrived.get((b, c), set()) == who:
            done.setdefault(b, set()).add(c)
    return count, done


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("full", [False, True])
def test_nobody_is_overtaken(backward, full):
    slots, progs = barriers(), programs(backward, full)
    count, _ = furthest(progs)
    assert all(count[n] == len(p) for n, p in progs.items())            # it ends
    waited = {b for p in progs.values() for _, b, _ in p}
    assert waited <= set(slots), waited - set(slots)
    late = []
    for n, p in progs.items():
        for at, (kind, b, c) in enumerate(p):
            if kind == "w" and c + slots[b] in furthest(progs, n, at)[1].get(b, set()):
                late.append((n, b, c))
    assert not late, late


@pytest.mark.parametrize("backward", [False, True])
def test_factors_stay_until_the_results_are_out(backward):
    """The warps that bring V in fetch the factors of the results of chunk i + 1 when they have handed on chunk i, into one of
    four buffers: not before chunk i - 3 is out."""
    progs = programs(backward, True)
    for at, (kind, b, c) in enumerate(progs["out"]):
        if (kind, b) == ("a", "x_free") and c + 3 < CHUNKS:
            handed_on = furthest(progs, "out", at)[1]["v_ready"]
            assert c + 3 not in handed_on, c
            assert backward or c + 2 in handed_on, c                         # three buffers would not do


def test_the_kernel_waits_by_slots():
    """A barrier of two phases is named with its slot wherever it is used."""
    text = open(SOURCE).read()
    for name, size in barriers().items():
        if size == 2:
            for use in re.findall(r"&%s\b(.)" % name, text):
                assert use == "[", name

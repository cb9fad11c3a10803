"""CPU test of the barriers of window attention's gradient pipeline: every wait goes by one
bit of a barrier's phase, so it is sound only if, while a warp stands at it, the phase before
the awaited one has passed and the one after cannot.  The steps of one tile are written down
as events with what must have happened before each; the ring depths, buffers and the indices
of the p_ready barriers are read from the kernel's source."""
import re
from collections import defaultdict

import pytest

from benchmark_b200 import build

SOURCE = (build.CSRC / "window_bwd_kernel.cuh").read_text()
STEPS = 30
QUADS, WARPS = 2, 2  # lane quadrants of the model, elementwise warps of each (all are alike)


def constant(name, keys, D):
    """TileCfg<D, keys>::name."""
    text = re.search(rf"static constexpr int {name} = (.+?);", SOURCE).group(1)
    text = re.sub(r"kKeys \? (\d+) : (\d+)", lambda m: m.group(1 if keys else 2), text)
    return eval(text.replace("/", "//"), {"D": D})


def p_ready_expressions():
    """The source's index of the p_ready barrier at step t, and what its phase bit is of."""
    assert "const int sb = t % C::kSBufs;  // S buffer" in SOURCE
    assert "const int buf = sb;" in SOURCE and "if (++sb == C::kSBufs) sb = 0;" in SOURCE
    wait = re.search(r"&p_ready\[([^\]]+)\], static_cast<uint32_t>\(([^)]+)\) & 1u", SOURCE)
    arrive = re.search(r"mbar_arrive_warp\(&p_ready\[([^\]]+)\]\)", SOURCE)
    at = {"sb": "t % C::kSBufs", "buf": "t % C::kSBufs"}
    index, other = (at.get(m.group(1), m.group(1)) for m in (wait, arrive))
    assert index == other
    return index, wait.group(2)


def faults(keys, D, index, phase):
    """Waits that one phase bit does not decide, and arrivals that could meet a phase that
    is not theirs."""
    n1, n2, bufs = (constant(c, keys, D) for c in ("kStages1", "kStages2", "kSBufs"))
    names = {"kSBufs": bufs}
    p_index = [eval(index.replace("C::", ""), dict(names, t=t)) for t in range(STEPS)]
    p_bit = [eval(phase.replace("C::", "").replace("/", "//"), dict(names, t=t)) & 1
             for t in range(STEPS)]
    after = defaultdict(set)   # event -> events that must come before it
    at, waits = [], []         # events; (at the wait, past it, barrier, phase)
    arrivals = defaultdict(list)  # (barrier, arriver) -> its arrivals in order
    bad = []                   # (barrier, phase, what)

    def event(*before):
        at.append(None)
        e = len(at) - 1
        after[e] |= set(b for b in before if b is not None)
        return e

    class Role:
        def __init__(self):
            self.last = None
            self.done = None  # last completion of its asynchronous work

        def wait(self, bar, m, bit=None):
            if m >= 0 and bit is not None and bit != m & 1:
                bad.append((bar, m, "bit"))
            here = event(self.last)
            self.last = event(here)
            waits.append((here, self.last, bar, m))

        def arrive(self, bar, who=0):
            self.last = event(self.last)
            arrivals[bar, who].append(self.last)

        def commit(self, bar):  # arrives when the work issued so far is complete
            self.last = event(self.last)
            self.done = event(self.last, self.done)
            arrivals[bar, 0].append(self.done)

    tma, issue, acc = Role(), Role(), Role()
    quads = [[Role() for _ in range(WARPS)] for _ in range(QUADS)]
    phases = defaultdict(int)  # of each p_ready barrier so far
    for t in range(STEPS):
        s1, s2, sb = t % n1, t % n2, t % bufs
        tma.wait(("empty1", s1), t // n1 - 1)
        tma.commit(("full1", s1))
        tma.done = None  # copies complete in any order
        tma.wait(("empty2", s2), t // n2 - 1)
        tma.commit(("full2", s2))
        tma.done = None
        issue.wait(("full1", s1), t // n1)
        issue.wait(("p_free", sb), t // bufs - 1)
        issue.wait(("full2", s2), t // n2)
        issue.wait(("dp_free",), t - 1)
        if not keys:
            issue.commit(("empty2", s2))
        issue.commit(("sd_ready",))
        for quad in quads:
            for w in quad:
                w.wait(("sd_ready",), t)
                if keys:
                    w.wait(("full2", s2), t // n2)
                w.arrive(("dp_free",), id(w))
            meet = event(*(w.last for w in quad))  # the quadrant's named barrier
            for w in quad:
                w.last = meet
                w.wait(("full1", s1), t // n1)  # rows that nothing sees are zeroed
                w.arrive(("p_ready", p_index[t]), id(w))
        acc.wait(("p_ready", p_index[t]), phases[p_index[t]], p_bit[t])
        phases[p_index[t]] += 1
        acc.commit(("empty1", s1))
        if keys:
            acc.commit(("empty2", s2))
        acc.commit(("p_free", sb))

    # A phase is complete with all of its arrivals; a wait is passed after its phase.
    by_bar = defaultdict(list)
    for (bar, _), events in arrivals.items():
        by_bar[bar].append(events)
    complete = {(bar, m): events for bar, lists in by_bar.items()
                for m, events in enumerate(zip(*lists))}
    for here, passed, bar, m in waits:
        if m >= 0:
            after[passed] |= set(complete[bar, m])
    # All that has happened before each event, as bits: earliest events first.
    left = {e: len(after[e]) for e in range(len(at))}
    then = defaultdict(list)
    for e in range(len(at)):
        for b in after[e]:
            then[b].append(e)
    past, ready = {}, [e for e, n in left.items() if n == 0]
    while ready:
        e = ready.pop()
        past[e] = sum({1 << b for b in after[e]}, 0)
        for b in after[e]:
            past[e] |= past[b]
        for x in then[e]:
            left[x] -= 1
            if left[x] == 0:
                ready.append(x)
    assert len(past) == len(at), "the steps wait for one another in a circle"

    def before(events, e):
        return all(past[e] >> x & 1 for x in events)
    for here, passed, bar, m in waits:
        if m >= 1 and not before(complete[bar, m - 1], here):
            bad.append((bar, m, "the phase before may not have passed"))
        after_it = complete.get((bar, m + 1))
        if after_it and not any(before([passed], e) for e in after_it):
            bad.append((bar, m, "the phase after may pass first"))
    for (bar, _), events in arrivals.items():
        for m, e in enumerate(events[1:]):
            if not before(complete[bar, m], e):
                bad.append((bar, m + 1, "an arrival may meet the phase before"))
    return bad


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [True, False])
def test_every_wait_is_decided_by_its_phase_bit(keys, D):
    assert faults(keys, D, *p_ready_expressions()) == []


def test_two_barriers_for_three_buffers_are_found():
    """The model itself: P of steps t and t + 2 on one barrier can both be ready before the
    accumulating warp looks, where three S buffers let the steps run that far ahead."""
    bad = faults(True, 128, "t & 1", "t >> 1")
    assert bad and all(b[0][0] == "p_ready" and "after" in b[2] for b in bad)
    assert faults(False, 128, "t & 1", "t >> 1") == []  # two buffers

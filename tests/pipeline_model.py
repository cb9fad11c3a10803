"""Model of a kernel's pipeline for CPU tests of its barriers.

A wait goes by one bit of a barrier's phase, so it is sound only if, while a warp stands
at it, the phase before the awaited one has passed and the one after cannot.  A pipeline
is written down as roles (warps) that wait, arrive and commit asynchronous work in order;
what must have happened before each of these events then decides every wait.
"""
from __future__ import annotations

from collections import defaultdict


class Role:
    """A warp: what it does, in order."""

    def __init__(self, pipeline):
        self.p = pipeline
        self.last = None
        self.done = None  # its last commit's arrival

    def wait(self, bar, phase, bit=None):
        """Wait for `phase` of `bar` (-1: none, passed at once) by the bit `bit`."""
        if phase >= 0 and bit is not None and bit != phase & 1:
            self.p.bad.append((bar, phase, "the bit is another phase's"))
        here = self.p.event(self.last)
        self.last = self.p.event(here)
        self.p.waits.append((here, self.last, bar, phase))

    def arrive(self, bar):
        self.last = self.p.event(self.last)
        self.p.arrivals[bar, id(self)].append(self.last)

    def commit(self, bar, in_order=False):
        """An arrival at some time after this, which nothing else waits for.  in_order: not
        before those of the role's earlier commits, which end with the same products."""
        self.last = self.p.event(self.last)
        done = self.p.event(self.last, self.done if in_order else None)
        self.done = done
        self.p.arrivals[bar, "async"].append(done)


class Pipeline:
    def __init__(self):
        self.before = []                   # per event, those that come before it
        self.waits = []                    # (at the wait, past it, barrier, phase)
        self.arrivals = defaultdict(list)  # (barrier, arriver) -> its arrivals in order
        self.bad = []                      # (barrier, phase, what)

    def role(self):
        return Role(self)

    def event(self, *before):
        self.before.append({b for b in before if b is not None})
        return len(self.before) - 1

    def meet(self, *roles):
        """A named barrier of these warps."""
        e = self.event(*(r.last for r in roles))
        for r in roles:
            r.last = e

    def faults(self):
        """(barrier, phase, what) of waits that one phase bit does not decide, and of
        arrivals that could meet a phase that is not theirs."""
        bad = list(self.bad)
        lists = defaultdict(list)
        for (bar, _), events in self.arrivals.items():
            lists[bar].append(events)
        # A phase is complete with all of its arrivals; a wait is passed after its phase.
        complete = {(bar, m): events for bar, each in lists.items()
                    for m, events in enumerate(zip(*each))}
        for _, passed, bar, m in self.waits:
            if m >= 0:
                self.before[passed] |= set(complete[bar, m])
        # All that has happened before each event, as bits: earliest events first.
        left = [len(b) for b in self.before]
        then = defaultdict(list)
        for e, earlier in enumerate(self.before):
            for b in earlier:
                then[b].append(e)
        past, ready = {}, [e for e, n in enumerate(left) if n == 0]
        while ready:
            e = ready.pop()
            past[e] = 0
            for b in self.before[e]:
                past[e] |= past[b] | 1 << b
            for x in then[e]:
                left[x] -= 1
                if left[x] == 0:
                    ready.append(x)
        assert len(past) == len(left), "the roles wait for one another in a circle"

        def are_before(events, e):
            return all(past[e] >> x & 1 for x in events)
        for here, passed, bar, m in self.waits:
            if m >= 1 and not are_before(complete[bar, m - 1], here):
                bad.append((bar, m, "the phase before may not have passed"))
            later = complete.get((bar, m + 1))
            if later and not any(are_before([passed], e) for e in later):
                bad.append((bar, m, "the phase after may pass first"))
        for (bar, _), events in self.arrivals.items():
            for m, e in enumerate(events[1:]):
                if not are_before(complete[bar, m], e):
                    bad.append((bar, m + 1, "an arrival may meet the phase before"))
        return bad

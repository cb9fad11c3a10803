"""CPU test of the barriers of window attention's gradient pipeline (pipeline_model): the
steps of a CTA's tiles, with the ring depths, buffers and the indices of the p_ready barriers read
from the kernel's source."""
import re
from collections import defaultdict

import pytest

import pipeline_model
from benchmark_b200 import build

SOURCE = (build.CSRC / "window_bwd_kernel.cuh").read_text()
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


def faults(keys, D, index, phase, items=(30,)):
    """Items of so many steps (those of a CTA; one that streams nothing is passed over)."""
    n1, n2, bufs = (constant(c, keys, D) for c in ("kStages1", "kStages2", "kSBufs"))
    index, phase = (x.replace("C::", "").replace("/", "//") for x in (index, phase))
    model = pipeline_model.Pipeline()
    tma, issue, acc = (model.role() for _ in range(3))
    quads = [[model.role() for _ in range(WARPS)] for _ in range(QUADS)]
    phases = defaultdict(int)  # of each p_ready barrier so far
    t = 0
    for li, steps in enumerate(n for n in items if n > 0):
        tma.wait(("own_empty",), li - 1)
        tma.commit(("own_full",))
        issue.wait(("own_full",), li)
        acc.wait(("acc_empty",), li - 1)
        for i in range(steps):
            s1, s2, sb = t % n1, t % n2, t % bufs
            at, bit = (eval(x, {"kSBufs": bufs, "t": t}) for x in (index, phase))
            tma.wait(("empty1", s1), t // n1 - 1)
            tma.commit(("full1", s1))
            tma.wait(("empty2", s2), t // n2 - 1)
            tma.commit(("full2", s2))
            issue.wait(("full1", s1), t // n1)
            issue.wait(("p_free", sb), t // bufs - 1)
            issue.wait(("full2", s2), t // n2)
            issue.wait(("dp_free",), t - 1)
            if not keys:
                issue.commit(("empty2", s2))
            issue.commit(("sd_ready",))
            if i + 1 == steps:
                issue.commit(("own_empty",))
            for quad in quads:
                for w in quad:
                    w.wait(("sd_ready",), t)
                    if keys:
                        w.wait(("full2", s2), t // n2)
                    w.arrive(("dp_free",))
                model.meet(*quad)
                for w in quad:
                    w.wait(("full1", s1), t // n1)  # rows that nothing sees are zeroed
                    w.arrive(("p_ready", at))
            acc.wait(("p_ready", at), phases[at], bit & 1)
            phases[at] += 1
            acc.commit(("empty1", s1))
            if keys:
                acc.commit(("empty2", s2))
            acc.commit(("p_free", sb))
            if i + 1 == steps:
                acc.commit(("acc_full",))
            t += 1
        for quad in quads:
            for w in quad:
                w.wait(("acc_full",), li)
                w.arrive(("acc_empty",))
    return model.faults()


@pytest.mark.parametrize("items", [(30,), (9, 0, 1, 4, 0, 0, 3, 1, 1, 2), (1,) * 8, (2,) * 6],
                         ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [True, False])
def test_every_wait_is_decided_by_its_phase_bit(keys, D, items):
    assert faults(keys, D, *p_ready_expressions(), items) == []


def test_two_barriers_for_three_buffers_are_found():
    """The model itself: P of steps t and t + 2 on one barrier can both be ready before the
    accumulating warp looks, where three S buffers let the steps run that far ahead."""
    bad = faults(True, 128, "t & 1", "t >> 1")
    assert bad and all(b[0][0] == "p_ready" and "after" in b[2] for b in bad)
    assert faults(False, 128, "t & 1", "t >> 1") == []  # two buffers

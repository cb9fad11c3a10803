"""CPU tests of the attention kernel's barriers (pipeline_model): items of several key
tiles, of one and of none (query rows before a request's first key)."""
import re
from collections import defaultdict

import pytest

import pipeline_model
from benchmark_b200 import build

SOURCE = (build.CSRC / "attention_kernel.cuh").read_text()
S_BUFS = int(re.search(r"constexpr int kSBufs = (\d+);", SOURCE).group(1))
WARPS = 2  # softmax and epilogue warps of the model (they are all alike)


def stages(name, D):
    """Cfg<D>'s ring depth."""
    m = re.search(rf"static constexpr int {name} = kPair \? \d+ : \(D == 128\) \? (\d+) : (\d+);",
                  SOURCE)
    return int(m.group(1 if D == 128 else 2))


def faults(items, D, skip=False):
    """Items of so many key tiles.  skip: the S issuer passes over items without any."""
    ks, vs = stages("kKStages", D), stages("kVStages", D)
    model = pipeline_model.Pipeline()
    tma_k, tma_v, issue_s, issue_pv = (model.role() for _ in range(4))
    softmax = [model.role() for _ in range(WARPS)]
    epilogue = [model.role() for _ in range(WARPS)]
    t, seen = 0, defaultdict(int)
    for li, n in enumerate(items):
        q = li & 1
        tma_k.wait(("q_empty", q), (li >> 1) - 1)
        tma_k.commit(("q_full", q))
        if n > 0 or not skip:
            issue_s.wait(("q_full", q), li >> 1)
        if n == 0:
            if skip:
                issue_pv.wait(("q_full", q), li >> 1)
            else:
                issue_s.arrive(("q_seen", q))
                issue_pv.wait(("q_seen", q), seen[q])
                seen[q] += 1
            issue_pv.wait(("o_empty",), li - 1)
        for j in range(n):
            sb = t % S_BUFS
            tma_k.wait(("k_empty", t % ks), t // ks - 1)
            tma_k.commit(("k_full", t % ks))
            tma_v.wait(("v_empty", t % vs), t // vs - 1)
            tma_v.commit(("v_full", t % vs))
            issue_s.wait(("k_full", t % ks), t // ks)
            issue_s.wait(("p_free", sb), t // S_BUFS - 1)
            issue_s.commit(("k_empty", t % ks), in_order=True)
            issue_s.commit(("s_ready", sb), in_order=True)
            for w in softmax:
                w.wait(("s_ready", sb), t // S_BUFS)
                if j > 0:  # a rescale
                    w.wait(("pv_done", (t - 1) & 1), (t - 1) >> 1)
                if vs < S_BUFS and t >= vs:  # rows of V are zeroed
                    w.wait(("pv_done", (t - vs) & 1), (t - vs) >> 1)
                w.wait(("v_full", t % vs), t // vs)
                w.arrive(("p_ready", sb))
            issue_pv.wait(("v_full", t % vs), t // vs)
            issue_pv.wait(("p_ready", sb), t // S_BUFS)
            if j == 0:
                issue_pv.wait(("o_empty",), li - 1)
            issue_pv.commit(("v_empty", t % vs), in_order=True)
            issue_pv.commit(("pv_done", t & 1), in_order=True)
            issue_pv.commit(("p_free", sb), in_order=True)
            t += 1
        issue_pv.commit(("o_full",), in_order=True)
        for w in softmax:
            w.wait(("o_empty",), li - 1)
            w.arrive(("l_ready", q))
        for w in epilogue:
            w.wait(("o_full",), li)
            w.wait(("l_ready", q), li >> 1)
            w.arrive(("o_empty",))
        model.meet(*epilogue)
        epilogue[0].arrive(("q_empty", q))
    return model.faults()


ITEMS = [[3] * 8, [1] * 10, [2, 1, 4, 1, 1], [0] * 6, [0, 0, 2, 0, 0, 3], [3, 0, 3, 0, 3],
         [0, 3, 0, 0, 0, 2, 1], [5, 0, 0, 0, 0, 1, 1, 0, 2]]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("items", ITEMS, ids=str)
def test_every_wait_is_decided_by_its_phase_bit(items, D):
    # What the model takes from the source: the S issuer waits for each item's Q first.
    flat = re.sub(r"\s+", " ", SOURCE)
    for text in ("++li; if (it.n == 0) { ok = warp_wait(&q_full[qb], qpar, kSiteQFull); "
                 "if (ok) mbar_arrive_warp(&q_seen[qb]); continue; } "
                 "ok = wait3(bar(&q_full[qb]), qpar, dn_a, dn_p, dn_a, dn_p, kSiteQFull);",
                 "ok = warp_wait(&q_seen[li & 1], (seen >> (li & 1)) & 1u, kSiteQFull) && "
                 "warp_wait(o_rd, oe_par, kSiteOEmpty);",
                 "commit_both(&pv_done[t & 1]); commit_lead(&p_free[sb]);"):
        assert text in flat
    assert faults(items, D) == []


def test_skipped_queries_are_found():
    """The model itself: after two items without key tiles the next one's Q could not be told
    from the first one's by the phase bit."""
    for D in (64, 128):
        bad = faults([0, 0, 2, 0, 0, 3], D, skip=True)
        assert bad and all(b[0][0] == "q_full" and "before" in b[2] for b in bad)
        assert faults([3, 0, 3, 0, 3], D, skip=True) == []

"""CPU tests of the two-Q-tile attention kernel: its barriers (pipeline_model), with units
of two query tiles and of one, and its registers."""
import re
import subprocess
from collections import defaultdict

import pytest

import pipeline_model
from benchmark_b200 import build

SOURCE = (build.CSRC / "attention_pair_kernel.cuh").read_text()
K_STAGES, V_STAGES = (int(re.search(rf"constexpr int {n} = (\d+);", SOURCE).group(1))
                      for n in ("kKStages", "kVStages"))
S_BUFS = int(re.search(r"constexpr int kSBufs = (\d+);",
                       (build.CSRC / "attention_kernel.cuh").read_text()).group(1))
WARPS = 2  # of a softmax pipe and of the epilogue in the model (all are alike)


def faults(units, tiles, shared=False):
    """Units of 1 or 2 query tiles over `tiles` key tiles.  shared: the scores of both pipes
    on one set of barriers."""
    model = pipeline_model.Pipeline()
    tma_k, tma_v, issue_s, issue_pv = (model.role() for _ in range(4))
    pipes = [[model.role() for _ in range(WARPS)] for _ in range(2)]
    epilogue = [model.role() for _ in range(WARPS)]
    seen = defaultdict(int)  # phases that a role has waited for

    def next_phase(role, bar):
        seen[id(role), bar] += 1
        return seen[id(role), bar] - 1

    t = u = 0
    lq = [0, 0]
    for nq in units:
        for pp in range(nq):
            q = (pp, lq[pp] & 1)
            tma_k.wait(("q_empty", *q), (lq[pp] >> 1) - 1)
            tma_k.commit(("q_full", *q))
            issue_s.wait(("q_full", *q), lq[pp] >> 1)
        u0 = u
        for j in range(tiles):
            ks, vs = t % K_STAGES, t % V_STAGES
            tma_k.wait(("k_empty", ks), t // K_STAGES - 1)
            tma_k.commit(("k_full", ks))
            tma_v.wait(("v_empty", vs), t // V_STAGES - 1)
            tma_v.commit(("v_full", vs))
            issue_s.wait(("k_full", ks), t // K_STAGES)
            for pp in range(nq):
                sb = u % S_BUFS
                p_ready = ("p_ready", pp, sb)
                s_ready = ("s_ready", sb) if shared else ("s_ready", pp, sb)
                issue_s.wait(("p_free", sb), u // S_BUFS - 1)
                issue_s.commit(s_ready)
                for w in pipes[pp]:
                    w.wait(s_ready, u // S_BUFS if shared else next_phase(w, s_ready))
                    if j > 0:  # a rescale waits for the pipe's tile before
                        prev = u - nq
                        w.wait(("p_free", prev % S_BUFS), prev // S_BUFS)
                    w.arrive(p_ready)
                issue_pv.wait(("v_full", vs), t // V_STAGES)
                issue_pv.wait(p_ready, next_phase(issue_pv, p_ready))
                if j == 0:
                    issue_pv.wait(("o_empty", pp), lq[pp] - 1)
                issue_pv.commit(("p_free", sb))
                u += 1
            issue_s.commit(("k_empty", ks))
            issue_pv.commit(("v_empty", vs))
            t += 1
        for pp in range(nq):
            issue_pv.commit(("o_full", pp))
            for w in pipes[pp]:
                w.wait(("o_empty", pp), lq[pp] - 1)
                w.arrive(("l_ready", pp))
            for w in epilogue:
                w.wait(("o_full", pp), lq[pp])
                w.wait(("l_ready", pp), lq[pp])
                w.arrive(("o_empty", pp))
            model.meet(*epilogue)
            epilogue[0].arrive(("q_empty", pp, lq[pp] & 1))
            lq[pp] += 1
        assert u == u0 + tiles * nq
    return model.faults()


UNITS = [[2] * 8, [1] * 12, [2, 1] * 6, [1, 2, 1, 1, 2, 2, 1], [2, 2, 1] * 4]


@pytest.mark.parametrize("tiles", [1, 2, 3, 5])
@pytest.mark.parametrize("units", UNITS, ids=str)
def test_every_wait_is_decided_by_its_phase_bit(units, tiles):
    # What the model takes from the source.
    for text in ("mma_commit_warp(&s_ready[pp * kSBufs + sb]);",
                 "warp_wait(&s_ready[pp * kSBufs + sb], (phases >> sb) & 1u, kSiteSReady);",
                 "const int pb = pp * kSBufs + sb;", "bar(&p_ready[pb]), (p_phase >> pb) & 1u,",
                 "mbar_arrive_warp(&p_ready[pp * kSBufs + sb]);",
                 "const int prev = uu - un.nq;", "&p_free[prev % kSBufs]"):
        assert text in SOURCE
    assert faults(units, tiles) == []


def test_barriers_that_both_pipes_share_are_found():
    """The model itself: the second pipe comes back from a unit with one query tile."""
    assert any(b[0][0] == "s_ready" for b in faults([2, 1] * 6, 3, shared=True))


def test_the_score_loop_keeps_its_registers(tmp_path):
    """Spills in the softmax warps' loop cost 2.7 % of the kernel's rate."""
    try:
        nvcc = build.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    src = tmp_path / "pair.cu"
    src.write_text('#include "attention_pair_kernel.cuh"\n'
                   "auto* kernel = &b200::attn::pair::attention_pair_kernel<1, false>;\n")
    out = subprocess.run([nvcc, "-Xptxas=-v", *build.ARCH, *build.COMMON, "-c", "-o",
                          str(tmp_path / "pair.o"), str(src)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    info = out.stdout + out.stderr
    spills = re.search(r"attention_pair_kernel.*?\n.*?(\d+) bytes spill stores, (\d+) bytes spill "
                       r"loads", info, flags=re.S)
    assert spills and spills.groups() == ("0", "0"), info

"""GPU tests of the attention layer's operators with NaN where queries look: each row that
sees it is NaN, its log-sum-exp too (-inf is a row that sees nothing), and no other row."""
import math

import pytest
import torch

import layer_util as U
from benchmark_b200 import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16

WINDOW = [  # B, Hq, Hkv, Sq, Skv, D, W, sinks
    (2, 32, 8, 1, 5000, 128, 1024, 4),     # 16-row tiles, a cluster of splits
    (1, 16, 8, 1, 8192, 64, 1 << 40, 0),   # many splits
    (40, 32, 16, 3, 200, 64, 150, 4),      # a unit to a warp
    (6, 8, 2, 300, 517, 128, 128, 4),      # 128-row tiles
    (4, 16, 4, 260, 1000, 64, 1 << 40, 0),
    (1, 32, 8, 600, 2000, 64, 700, 20),
    (1, 8, 2, 200, 9000, 128, 1 << 40, 0),  # their keys split
    (2, 12, 4, 333, 7000, 64, 1 << 40, 0),
]


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(BF16)


def inputs(case, at):
    """q, k, v with one NaN among each head's keys, and the rows [B, Hq, Sq] that see it."""
    B, Hq, Hkv, Sq, Skv, D, W, sinks = case
    g = torch.Generator(device="cuda").manual_seed(at)
    q, k, v = randn(g, B, Hq, Sq, D), randn(g, B, Hkv, Skv, D), randn(g, B, Hkv, Skv, D)
    first = max(0, Skv - Sq - min(W, Skv) + 1)  # the keys that some query may see
    j = first + (torch.arange(B * Hkv, device="cuda").view(B, Hkv) * 37 + at) % (Skv - first)
    clean = k.clone()
    k.scatter_(2, j[:, :, None, None], math.nan)  # column 0 of key j
    seen = U.visible(torch.full((B,), Skv, device="cuda"), Sq, Skv, W, sinks, "cuda")
    heads = j.repeat_interleave(Hq // Hkv, dim=1)[:, :, None, None].expand(B, Hq, Sq, 1)
    hit = seen.expand(B, Hq, Sq, Skv).gather(3, heads).squeeze(3)
    return q, k, v, clean, hit


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_lse_of_a_row_that_sees_nan(case):
    B, Hq, _, Sq, _, _, W, sinks = case
    for at in (0, 5, 40):
        q, k, v, clean, hit = inputs(case, at)
        lse, want = (torch.empty((B, Hq, Sq), device="cuda") for _ in range(2))
        o = ops.attention_window_fwd(q, k, v, W, sinks, lse=lse)
        ops.attention_window_fwd(q, clean, v, W, sinks, lse=want)
        ops.check()
        assert hit.any() and torch.isnan(lse[o.isnan().any(-1)]).all()
        assert torch.equal(lse[~hit], want[~hit])


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_rows_that_see_nan(case):
    """At head_dim 64 a part of the exponentials goes by a polynomial."""
    W, sinks = case[6:]
    for at in range(0, 64, 7):
        q, k, v, clean, hit = inputs(case, at)
        o = ops.attention_window_fwd(q, k, v, W, sinks)
        want = ops.attention_window_fwd(q, clean, v, W, sinks)
        ops.check()
        assert o[hit].isnan().all() and torch.equal(o[~hit], want[~hit])


@pytest.mark.parametrize("B,Hq,Hkv,Sq,P,S", [(40, 16, 16, 1, 5003, 20), (3, 16, 4, 1, 517, 128)])
@pytest.mark.parametrize("D", [64, 128])
def test_prefix_with_nan(B, Hq, Hkv, Sq, P, S, D):
    g = torch.Generator(device="cuda").manual_seed(1)
    q, kp, vp = randn(g, B, Hq, Sq, D), randn(g, Hkv, P, D), randn(g, Hkv, P, D)
    k, v = randn(g, B, Hkv, S, D), randn(g, B, Hkv, S, D)
    want = ops.attention_shared_prefix(q, kp, vp, k, v)
    for at in range(0, 64, 7):
        x = kp.clone()
        x[Hkv // 2, (at * 71) % P, 3] = math.nan
        o = ops.attention_shared_prefix(q, x, vp, k, v)
        ops.check()
        hit = torch.arange(Hq, device="cuda") // (Hq // Hkv) == Hkv // 2
        assert o[:, hit].isnan().all() and torch.equal(o[:, ~hit], want[:, ~hit])


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_queries_that_hold_nan(case):
    B, Hq, Hkv, Sq, Skv, D, W, sinks = case
    q, k, v, clean, _ = inputs(case, 3)
    hit = torch.rand((B, Hq, Sq), generator=torch.Generator(device="cuda").manual_seed(3),
                     device="cuda") < 0.2
    x = q.clone()
    x[..., 5] = torch.where(hit, torch.tensor(math.nan, dtype=BF16, device="cuda"), x[..., 5])
    lse, want_lse = (torch.empty((B, Hq, Sq), device="cuda") for _ in range(2))
    o = ops.attention_window_fwd(x, clean, v, W, sinks, lse=lse)
    want = ops.attention_window_fwd(q, clean, v, W, sinks, lse=want_lse)
    ops.check()
    assert o[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(o[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])

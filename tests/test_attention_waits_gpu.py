"""GPU tests of the attention kernels where a softmax warp runs ahead of the matrix
products: keys that equal the queries raise most rows' maxima late and by much, so that
accumulators are rescaled often, between many work units per SM.  Results against the
plain 64-bit form (layer_util, which derives the tolerances), and equal call by call."""
import pytest
import torch

import layer_util as U
from benchmark_b200 import ops

pytestmark = pytest.mark.gpu


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def check(call, want, bound, repeats=20):
    first = call()
    assert ((first[:want.shape[0]].double() - want).abs() <= bound).all()
    for _ in range(repeats):
        assert torch.equal(call(), first)
    ops.check()


def inputs(seed, B, H, S, D):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return randn(g, B, H, S, D), randn(g, B, H, S, D)


def form(k, v, B, window=None, sinks=0):
    """The plain form of the first B requests, the keys as queries."""
    S = k.shape[2]
    if window is None:
        seen = torch.ones(B, 1, S, S, dtype=torch.bool, device="cuda")
    else:
        seen = U.visible(torch.full((B,), S, device="cuda"), S, S, window, sinks, "cuda")
    want, bound, _, _ = U.attention(k[:B], k[:B], v[:B], seen)
    return want, bound


@pytest.mark.parametrize("B,H,S,D,causal", [
    (64, 2, 600, 128, True), (64, 2, 600, 128, False), (16, 8, 1000, 128, True),
    (4, 32, 2048, 128, False), (64, 2, 600, 64, True), (4, 32, 2048, 64, True),
])
def test_rescales_wait_for_the_previous_product(B, H, S, D, causal):
    """A rescale waits for the product of the tile before; the one before that may not
    have completed either."""
    k, v = inputs(30, B, H, S, D)
    want, bound = form(k, v, 1, S if causal else None)
    check(lambda: ops.attention_fwd(k, k, v, causal=causal), want, bound)


@pytest.mark.parametrize("D", [64, 128])
def test_zeroed_values_wait_for_the_products_before(D):
    """Rows of V that no query of a tile may see are zeroed in the tile's stage, once the
    products that read the stage before have completed."""
    B, H, S, window, sinks = 32, 4, 1100, 200, 3
    k, v = inputs(31, B, H, S, D)
    want, bound = form(k, v, 1, window, sinks)
    check(lambda: ops.attention_window_fwd(k, k, v, window, sinks), want, bound)


@pytest.mark.parametrize("B,H,S", [(64, 2, 600), (64, 2, 640), (64, 2, 768), (200, 1, 130),
                                   (300, 2, 128), (64, 4, 384)])
def test_pairs_of_query_tiles_with_one_left_over(B, H, S):
    """head_dim 64, not causal: with an odd number of query tiles one of the two softmax
    pipes sits out every unit that has only one."""
    k, v = inputs(32, B, H, S, 64)
    want, bound = form(k, v, B)
    check(lambda: ops.attention_fwd(k, k, v), want, bound)

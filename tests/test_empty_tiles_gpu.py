"""GPU tests of attention over many query tiles that see no key, between others that do:
requests shorter than their queries.  Queries come from memory, keys that many tiles share
from L2."""
import pytest
import torch

import layer_util as U
from benchmark_b200 import ops

pytestmark = pytest.mark.gpu


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def check(call, want, bound):
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = call()
    U.check_close(first, want, bound, "o")
    for _ in range(5):
        flush.zero_()
        assert torch.equal(call(), first)
    ops.check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Skv", [40, 130, 500])
def test_causal_with_more_queries_than_keys(D, Skv):
    g = torch.Generator(device="cuda").manual_seed(40)
    B, Hq, Hkv, Sq = 40, 8, 2, 1024
    q, k, v = randn(g, B, Hq, Sq, D), randn(g, B, Hkv, Skv, D), randn(g, B, Hkv, Skv, D)
    seen = U.visible(torch.full((B,), Skv, device="cuda"), Sq, Skv, Skv, 0, "cuda")
    want, bound, _, _ = U.attention(q, k, v, seen)
    check(lambda: ops.attention_fwd(q, k, v, causal=True), want, bound)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [(0, 0, 700), (1, 130, 700, 300), (129, 0), (0, 0, 0, 0, 511)],
                         ids=str)
def test_window_of_requests_shorter_than_their_queries(D, lens):
    g = torch.Generator(device="cuda").manual_seed(41)
    B, Hq, Hkv, Sq, Skv, W, sinks = 60, 8, 2, 512, 700, 200, 3
    q, k, v = randn(g, B, Hq, Sq, D), randn(g, B, Hkv, Skv, D), randn(g, B, Hkv, Skv, D)
    n = torch.tensor([lens[i % len(lens)] for i in range(B)], dtype=torch.int32, device="cuda")
    seen = U.visible(n, Sq, Skv, W, sinks, "cuda")
    want, bound, _, _ = U.attention(q, k, v, seen)
    check(lambda: ops.attention_window_fwd(q, k, v, W, sinks, kv_len=n), want, bound)


@pytest.mark.parametrize("D", [64, 128])
def test_keys_split_where_some_splits_see_none(D):
    g = torch.Generator(device="cuda").manual_seed(42)
    B, Hq, Hkv, Sq, Skv = 3, 8, 2, 260, 9000
    q, k, v = randn(g, B, Hq, Sq, D), randn(g, B, Hkv, Skv, D), randn(g, B, Hkv, Skv, D)
    n = torch.tensor([30, 200, 300], dtype=torch.int32, device="cuda")
    seen = U.visible(n, Sq, Skv, 1 << 40, 0, "cuda")
    want, bound, _, _ = U.attention(q, k, v, seen)
    check(lambda: ops.attention_window_fwd(q, k, v, 1 << 40, kv_len=n), want, bound)

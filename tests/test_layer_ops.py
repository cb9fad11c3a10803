"""CPU tests of the attention layer's operators: what their entry points refuse, what
their workspaces need, and the plain forms' gradients against differences."""
import ctypes
import math

import pytest
import torch

import layer_util as U
from benchmark_b200 import _lib, ops


def T(data=256, sb=8 * 1024 * 128, sh=1024 * 128, ss=128):
    return _lib.Tensor(data, sb, sh, ss)


def window(q=None, k=None, v=None, o=None, B=2, Hq=8, Hkv=2, Sq=64, Skv=1024, D=128, W=256,
           sinks=4, scale=-1.0, ws=256, ws_bytes=1 << 40):
    t = [T() if x is None else x for x in (q, k, v, o)]
    return _lib.lib().attention_window_fwd(*t, None, None, B, Hq, Hkv, Sq, Skv, D, W, sinks, scale,
                                           ws, ws_bytes, None)


@pytest.mark.parametrize("bad,status,word", [
    (dict(q=T(0)), 1, "null"), (dict(k=T(24)), 1, "aligned"), (dict(v=T(ss=129)), 1, "multiples"),
    (dict(k=T(sh=-8)), 1, "negative"), (dict(o=T(sh=0)), 1, "overlap"),
    (dict(o=T(ss=64)), 1, "overlap"), (dict(o=T(sb=1024)), 1, "overlap"),
    (dict(k=T(ss=0)), 1, "share a row"), (dict(q=T(sb=1 << 39)), 2, "2^39"), (dict(B=0), 1, "shape"), (dict(Sq=0), 1, "shape"),
    (dict(Skv=0), 1, "shape"), (dict(Hq=7), 1, "Hkv"), (dict(D=96), 2, "head_dim"),
    (dict(W=0), 1, "window"), (dict(sinks=-1), 1, "sinks"), (dict(scale=math.inf), 1, "scale"),
    (dict(scale=math.nan), 1, "scale"), (dict(Skv=(1 << 30) + 1), 2, "2^30"),
])
def test_window_refuses(bad, status, word):
    assert window(**bad) == status
    assert word in _lib.last_error()


def test_window_needs_its_workspace():
    n = ctypes.c_size_t()
    L = _lib.lib()
    assert L.attention_window_fwd_workspace(1, 8, 2, 1, 4096, 128, 4096, 0, ctypes.byref(n)) == 0
    assert n.value > 0
    args = dict(B=1, Sq=1, Skv=4096, W=4096, sinks=0)
    assert window(**args, ws=None, ws_bytes=0) == _lib.B200_EINVAL
    assert "workspace" in _lib.last_error()
    assert window(**args, ws_bytes=n.value - 1) == _lib.B200_EINVAL
    assert window(**args, ws=264) == _lib.B200_EINVAL  # not 16-byte aligned
    # Many rows need none.
    assert L.attention_window_fwd_workspace(4, 32, 8, 4096, 4096, 128, 512, 0,
                                            ctypes.byref(n)) == 0
    assert n.value == 0
    assert L.attention_window_fwd_workspace(1, 8, 3, 1, 4096, 128, 1, 0, ctypes.byref(n)) == 1
    assert L.attention_window_fwd_workspace(1, 8, 2, 1, 4096, 128, 1, 0, None) == 1


def window_bwd(B=2, Hq=8, Hkv=2, Sq=64, Skv=1024, D=128, W=256, sinks=4, lse=256, ws=256,
               ws_bytes=1 << 40, **over):
    names = ("dout", "q", "k", "v", "o", "dq", "dk", "dv")
    t = {n: over.get(n, T()) for n in names}
    return _lib.lib().attention_window_bwd(t["dout"], t["q"], t["k"], t["v"], t["o"], lse, t["dq"],
                                           t["dk"], t["dv"], None, B, Hq, Hkv, Sq, Skv, D, W,
                                           sinks, -1.0, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,status,word", [
    (dict(dout=T(0)), 1, "dout"), (dict(o=T(8)), 1, "o must"), (dict(dq=T(ss=0)), 1, "dq"),
    (dict(dk=T(sh=128)), 1, "dk"), (dict(dv=T(sb=-8)), 1, "dv"), (dict(lse=None), 1, "lse"),
    (dict(D=32), 2, "head_dim"), (dict(W=-1), 1, "window"), (dict(ws=None), 1, "workspace"),
    (dict(ws_bytes=100), 1, "too small"),
])
def test_window_bwd_refuses(bad, status, word):
    assert window_bwd(**bad) == status
    assert word in _lib.last_error()


def test_window_bwd_workspace():
    L, n = _lib.lib(), ctypes.c_size_t()

    def need(Sq, W, sinks):
        assert L.attention_window_bwd_workspace(1, 8, 2, Sq, Sq, 128, W, sinks,
                                                ctypes.byref(n)) == 0
        return n.value
    # Two floats for each query, padded to 64; sums of the sinks' parts where they are divided.
    assert need(100, 100, 0) == need(128, 128, 0) == 2 * 4 * 8 * 128
    assert need(4096, 64, 4) > need(4096, 64, 0) == 2 * 4 * 8 * 4096
    assert L.attention_window_bwd_workspace(1, 8, 2, 0, 1, 128, 1, 0, ctypes.byref(n)) == 1
    assert L.attention_window_bwd_workspace(1, 8, 2, 1, 1, 128, 1, 0, None) == 1


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv", [
    (1 << 10, 1 << 20, 1 << 20, 1 << 30, 1 << 30), (1, 1 << 10, 1, 1 << 20, 1 << 30),
    (1 << 30, 1, 1, 1 << 30, 1 << 30), (1, 1, 1, 1, 1 << 30)])
def test_workspaces_of_the_largest_shapes(B, Hq, Hkv, Sq, Skv):
    """The plans of shapes that no memory holds are formed without overflow."""
    L, n = _lib.lib(), ctypes.c_size_t()
    for window in (1, 1 << 30):
        args = (B, Hq, Hkv, Sq, Skv, 128, window, 4, ctypes.byref(n))
        assert L.attention_window_fwd_workspace(*args) == 0 and n.value < 1 << 30
        assert L.attention_window_bwd_workspace(*args) == 0
        assert n.value >= 8 * B * Hq * Sq


def rope(q=None, k=None, qo=None, ko=None, wq=256, wk=256, freq=256, R=128, pos=256, pos_sb=0,
         eps=1e-6, B=2, S=16, Hq=8, Hkv=2, D=128):
    t = [T() if x is None else x for x in (q, k, qo, ko)]
    return _lib.lib().qk_norm_rope(t[0], t[1], wq, wk, 0, freq, R, 0, pos, pos_sb, eps, t[2], t[3],
                                   B, S, Hq, Hkv, D, None)


@pytest.mark.parametrize("bad,status,word", [
    (dict(q=T(0)), 1, "q"), (dict(ko=T(ss=8)), 1, "k_out"), (dict(k=T(ss=12)), 1, "k"),
    (dict(wq=None), 1, "weight"), (dict(wk=260), 1, "weights must"), (dict(freq=None), 1, "inv_freq"), (dict(pos=None), 1, "positions"),
    (dict(R=24), 2, "rotary_dim"), (dict(R=144), 2, "rotary_dim"), (dict(R=-16), 2, "rotary_dim"),
    (dict(eps=-1.0), 1, "eps"), (dict(eps=math.nan), 1, "eps"), (dict(D=80), 2, "head_dim"),
    (dict(S=0), 1, "shape"), (dict(pos_sb=-1), 1, "stride"), (dict(S=1 << 30), 2, "tokens"),
    (dict(Hkv=(1 << 20) + 1), 2, "heads"),
])
def test_norm_rope_refuses(bad, status, word):
    assert rope(**bad) == status
    assert word in _lib.last_error()


def test_norm_rope_bwd_refuses():
    L = _lib.lib()
    n = ctypes.c_size_t()
    assert L.qk_norm_rope_bwd_workspace(2, 16, 128, ctypes.byref(n)) == 0 and n.value > 0
    assert L.qk_norm_rope_bwd_workspace(0, 16, 128, ctypes.byref(n)) == 1

    def bwd(dw=256, ws=256, ws_bytes=n.value, dq=None):
        t = T()
        return L.qk_norm_rope_bwd(t, t, t, t, 256, 256, 0, 256, 128, 0, 256, 0, 1e-6, dq or t, t,
                                  dw, dw, 2, 16, 8, 2, 128, ws, ws_bytes, None)
    assert bwd(dw=None) == 1 and "weight gradient" in _lib.last_error()
    assert bwd(ws=None) == 1 and "workspace" in _lib.last_error()
    assert bwd(ws_bytes=16) == 1 and "too small" in _lib.last_error()
    assert bwd(dq=T(ss=8)) == 1 and "dq" in _lib.last_error()


@pytest.mark.parametrize("B,S,D,status,word", [
    (2, 16, -1, 2, "head_dim"), (2, 16, 0, 2, "head_dim"), (2, 16, 96, 2, "head_dim"),
    (2, 0, 128, 1, "shape"), (-1, 16, 128, 1, "shape"),
])
def test_norm_rope_bwd_workspace_refuses(B, S, D, status, word):
    n = ctypes.c_size_t()
    assert _lib.lib().qk_norm_rope_bwd_workspace(B, S, D, ctypes.byref(n)) == status
    assert word in _lib.last_error()
    assert _lib.lib().qk_norm_rope_bwd_workspace(2, 16, 128, None) == 1


def prefix(P=4096, B=4, Hq=8, Hkv=2, Sq=1, S=64, D=128, kp=None, vp=None, k=None, o=None, ws=256,
           ws_bytes=1 << 40):
    t = T()
    return _lib.lib().attention_shared_prefix(t, kp or t, vp or t, k or t, t, o or t, None, B, Hq,
                                              Hkv, Sq, P, S, D, -1.0, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,status,word", [
    (dict(P=-1), 1, "prefix length"), (dict(S=0), 1, "shape"), (dict(D=256), 2, "head_dim"),
    (dict(kp=T(0)), 1, "k_prefix"), (dict(vp=T(ss=4)), 1, "v_prefix"), (dict(k=T(8)), 1, "k must"),
    (dict(o=T(sh=0)), 1, "overlap"), (dict(ws=None), 1, "workspace"),
    (dict(ws_bytes=64), 1, "too small"), (dict(Hkv=3), 1, "Hkv"),
])
def test_prefix_refuses(bad, status, word):
    assert prefix(**bad) == status
    assert word in _lib.last_error()


def test_python_refuses_cpu_tensors():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.attention_window_fwd(q, q, q, 4)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, q, q[0, 0, 0], q[0, 0, 0], torch.ones(8), torch.zeros(4))


def test_python_refuses_a_stream_of_another_device():
    class Stream:
        device = torch.device("cuda", 1)
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        ops.attention_window_fwd(q, q, q, 4, stream=Stream())


def directional(f, inputs, grads, seed=0, h=1e-5):
    """The gradients' inner product with a direction, and f's difference along it."""
    g = torch.Generator().manual_seed(seed)
    d = [torch.randn(x.shape, generator=g, dtype=U.F64) for x in inputs]
    diff = (f(*[x + h * u for x, u in zip(inputs, d)])
            - f(*[x - h * u for x, u in zip(inputs, d)])) / (2 * h)
    return sum((a * u).sum() for a, u in zip(grads, d)).item(), diff.item()


@pytest.mark.parametrize("interleaved", [False, True])
def test_plain_norm_rope_gradient_is_its_difference(interleaved):
    g = torch.Generator().manual_seed(1)
    x, gy = (torch.randn(2, 3, 5, 64, generator=g, dtype=U.F64) for _ in range(2))
    w = torch.randn(64, generator=g, dtype=U.F64)
    angles = U.rope_angles(torch.arange(5), torch.rand(16, generator=g, dtype=U.F64), 2)
    dx, _, dw, _ = U.norm_rope_bwd(gy, x, w, angles, 1e-3, interleaved)
    got, diff = directional(lambda a, b: (U.norm_rope(a, b, angles, 1e-3, interleaved)[0]
                                          * gy).sum(), (x, w), (dx, dw))
    assert got == pytest.approx(diff, rel=1e-7)


def test_plain_attention_gradient_is_its_difference():
    g = torch.Generator().manual_seed(2)
    q, do = (torch.randn(2, 4, 7, 16, generator=g, dtype=U.F64) for _ in range(2))
    k, v = (torch.randn(2, 2, 11, 16, generator=g, dtype=U.F64) for _ in range(2))
    seen = U.visible(torch.tensor([11, 5]), 7, 11, 4, 2, "cpu")  # rows that see nothing too
    o, _, lse, _ = U.attention(q, k, v, seen)
    grads = [t for t, _ in U.attention_bwd(do, q, k, v, o, lse, seen)]
    got, diff = directional(lambda a, b, c: (U.attention(a, b, c, seen)[0] * do).sum(), (q, k, v),
                            grads)
    assert got == pytest.approx(diff, rel=1e-7)

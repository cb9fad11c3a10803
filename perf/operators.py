"""Cases that measure the attention-layer operators: query/key norm with position
rotation, attention with a sliding window and sink tokens (both forward and
backward), and attention over a prefix that a whole batch shares.

With `own` false, `run` computes an operator in its plain form: elementary torch
operations in 32 bits (angles and long sums in 64), rounded once at the end.  With
`own` true it makes the call that a user of this package makes.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
NEG = float("-inf")
EPS = 1e-6


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One new token of one request, before its key enters the cache: latency.
        dict(name="norm_rope_1_token", op="norm_rope", B=1, S=1, Hq=32, Hkv=8, D=128, R=128,
             interleaved=False, wbits=16, far=30000),
        # A full training/prefill step's tokens, read from the fused projection's output.
        dict(name="norm_rope_4x4096", op="norm_rope", B=4, S=4096, Hq=32, Hkv=8, D=128, R=128,
             interleaved=False, wbits=32, far=4096),
        # The gradients of that step.
        dict(name="norm_rope_bwd_4x4096", op="norm_rope_bwd", B=4, S=4096, Hq=32, Hkv=8, D=128,
             R=128, interleaved=False, wbits=32, far=4096),
        # A short odd batch, head size 64, half of it rotated, adjacent pairs: the weights'
        # gradients weigh most here.
        dict(name="norm_rope_bwd_odd", op="norm_rope_bwd", B=2, S=333, Hq=10, Hkv=5, D=64, R=32,
             interleaved=True, wbits=16, far=200000),
        # Prefill of a sliding-window layer.
        dict(name="window_prefill_8192", op="window", B=1, Hq=32, Hkv=8, Sq=8192, Skv=8192, D=128,
             W=1024, sinks=4, lens="full"),
        # A padded batch's chunk behind its caches: other lengths in each row of it.
        dict(name="window_chunk_odd", op="window", B=3, Hq=12, Hkv=4, Sq=777, Skv=2500, D=64,
             W=300, sinks=5, lens="mixed"),
        # One token of one request: latency.
        dict(name="window_decode_1", op="window", B=1, Hq=32, Hkv=8, Sq=1, Skv=2048, D=128,
             W=1024, sinks=4, lens="mixed"),
        # A serving batch's tokens over caches longer than the window.
        dict(name="window_decode_64", op="window", B=64, Hq=64, Hkv=8, Sq=1, Skv=8192, D=128,
             W=4096, sinks=4, lens="mixed"),
        # The gradients of a training step's sliding-window layer.
        dict(name="window_bwd_4096", op="window_bwd", B=2, Hq=32, Hkv=8, Sq=4096, Skv=4096, D=128,
             W=1024, sinks=4, lens="full"),
        # A padded batch's chunk: other lengths in each row of it, a head for each query.
        dict(name="window_bwd_odd", op="window_bwd", B=3, Hq=6, Hkv=6, Sq=777, Skv=1001, D=64,
             W=300, sinks=5, lens="mixed"),
        # Three requests behind a short system text: latency.
        dict(name="prefix_3", op="prefix", B=3, Hq=16, Hkv=4, Sq=1, P=517, S=128, D=64,
             lens="mixed"),
        # A serving batch behind a long document.
        dict(name="prefix_64", op="prefix", B=64, Hq=64, Hkv=8, Sq=1, P=16384, S=1024, D=128,
             lens="mixed"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope_bwd", "window", "window", "window_bwd", "prefix",
                     "prefix"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    Hq = min(64, Hkv * group) // Hkv * Hkv
    if op in ("norm_rope", "norm_rope_bwd"):
        B = _spread(rng, 1, 32)
        most = 4 * 4096 * 40 * 128 // ((Hq + Hkv) * D)
        S = _spread(rng, 1, max(1, min(16384, most // B)))
        return dict(op=op, B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, R=rng.choice([16, 32, D // 2, D, D]),
                    interleaved=rng.random() < 0.5, wbits=rng.choice([16, 32]),
                    far=_spread(rng, 100, 1000000))
    if op in ("window", "window_bwd"):
        back = op == "window_bwd"
        while True:
            B = _spread(rng, 1, 16 if back else 64)
            # (With one key the scores' gradients are exact zeros, which says nothing.)
            Skv = _spread(rng, 32, 8192) if back else _spread(rng, 1, 16384)
            if rng.random() < 0.5:
                Sq = Skv if back else rng.choice([1, 1, 1, 2, 4, 8])
            else:
                Sq = _spread(rng, 1, 8192)
            # The dense scores of the plain form, and the caches, within the listed cases'.
            if (Sq <= Skv and B * Hq * Sq * Skv <= (64 * 4096 * 4096 if back else 32 * 8192 * 8192)
                    and B * Hkv * Skv * D <= 64 * 8 * 8192 * 128):
                break
        W = _spread(rng, 16, 8192)
        case = dict(op=op, B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, Skv=Skv, D=D, W=W,
                    sinks=rng.choice([0, 1, 4, 4, 16, 100, 130]),
                    lens=rng.choice(["full", "mixed", "mixed"]))
        while work(case)["flops"] > 4 * 128 * 32 * 8192 * 1028:
            case["W"] = max(16, case["W"] // 2)
            case["sinks"] = min(case["sinks"], 4)
        return case
    while True:
        B = _spread(rng, 1, 256)
        P = _spread(rng, 1, 32768)
        S = _spread(rng, 1, 4096)
        Sq = min(S, rng.choice([1, 1, 1, 2, 4]))
        if (B * Hkv * S * D <= 64 * 8 * 1024 * 128 and Hkv * P * D <= 8 * 16384 * 128
                and B * Hq * Sq * P * D <= 64 * 64 * 16384 * 128 and Hq // Hkv * Sq <= 64):
            break
    return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, Sq=Sq, P=P, S=S, D=D,
                lens=rng.choice(["full", "mixed", "mixed"]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(BF16)


def _lens(case, g, most, least):
    """The requests' cache lengths: all full, or spread over [least, most]."""
    if case["lens"] == "full":
        return torch.full((case["B"],), most, dtype=torch.int32, device="cuda")
    return torch.randint(least, most + 1, (case["B"],), generator=g, device="cuda",
                         dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": dict(case)}
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    if case["op"] in ("norm_rope", "norm_rope_bwd"):
        S = case["S"]
        # The fused projection's output [B, S, heads, D]; q and k are views of it.
        qkv = _normal(g, B, S, Hq + 2 * Hkv, D, scale=1.7)
        st["q"] = qkv[:, :, :Hq].transpose(1, 2)
        st["k"] = qkv[:, :, Hq:Hq + Hkv].transpose(1, 2)
        wt = BF16 if case["wbits"] == 16 else F32
        for n in ("wq", "wk"):
            st[n] = (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(wt)
        i = torch.arange(case["R"] // 2, dtype=F64)
        st["inv_freq"] = (10000.0 ** (-2.0 * i / case["R"])).to(F32).cuda()
        first = torch.randint(0, case["far"], (B, 1), generator=g, device="cuda")
        st["pos"] = (first + torch.arange(S, device="cuda")).to(torch.int32)
        if case["op"] == "norm_rope_bwd":
            st["gq"] = _normal(g, B, Hq, S, D, scale=0.3)
            st["gk"] = _normal(g, B, Hkv, S, D, scale=0.3)
        return st
    Sq = case["Sq"]
    st["q"] = _normal(g, B, Hq, Sq, D)
    if case["op"] in ("window", "window_bwd"):
        st["k"] = _normal(g, B, Hkv, case["Skv"], D)
        st["v"] = _normal(g, B, Hkv, case["Skv"], D)
        # Some rows of a padded batch may be shorter than the queries: their first rows see nothing.
        st["len"] = _lens(case, g, case["Skv"], max(1, case["Skv"] // 2))
        if case["op"] == "window_bwd":  # what the forward pass left, and the output's gradient
            st["o"], st["lse"] = _window(st["q"], st["k"], st["v"], st["len"], case["W"],
                                         case["sinks"])
            st["do"] = _normal(g, B, Hq, Sq, D, scale=0.5)
    else:
        st["kp"] = _normal(g, Hkv, case["P"], D)
        st["vp"] = _normal(g, Hkv, case["P"], D)
        st["k"] = _normal(g, B, Hkv, case["S"], D)
        st["v"] = _normal(g, B, Hkv, case["S"], D)
        st["len"] = _lens(case, g, case["S"], min(Sq, case["S"]))
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if own:
        from benchmark_b200 import ops
        if c["op"] == "norm_rope":
            return ops.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["inv_freq"],
                                    st["pos"], eps=EPS, interleaved=c["interleaved"])
        if c["op"] == "norm_rope_bwd":
            return ops.qk_norm_rope_bwd(st["gq"], st["gk"], st["q"], st["k"], st["wq"], st["wk"],
                                        st["inv_freq"], st["pos"], eps=EPS,
                                        interleaved=c["interleaved"])
        if c["op"] == "window":
            return ops.attention_window_fwd(st["q"], st["k"], st["v"], c["W"], c["sinks"],
                                            kv_len=st["len"])
        if c["op"] == "window_bwd":
            return ops.attention_window_bwd(st["do"], st["q"], st["k"], st["v"], st["o"],
                                            st["lse"], c["W"], c["sinks"], kv_len=st["len"])
        return ops.attention_shared_prefix(st["q"], st["kp"], st["vp"], st["k"], st["v"],
                                           kv_len=st["len"])
    if c["op"] == "norm_rope":
        cos, sin = _angles(st)
        return (_norm_rope(st["q"], st["wq"], cos, sin, c["interleaved"]),
                _norm_rope(st["k"], st["wk"], cos, sin, c["interleaved"]))
    if c["op"] == "norm_rope_bwd":
        cos, sin = _angles(st)
        dq, dwq = _norm_rope_bwd(st["gq"], st["q"], st["wq"], cos, sin, c["interleaved"])
        dk, dwk = _norm_rope_bwd(st["gk"], st["k"], st["wk"], cos, sin, c["interleaved"])
        return dq, dk, dwq, dwk
    if c["op"] == "window":
        return _window(st["q"], st["k"], st["v"], st["len"], c["W"], c["sinks"])[0]
    if c["op"] == "window_bwd":
        return _window_bwd(st["do"], st["q"], st["k"], st["v"], st["o"], st["lse"], st["len"],
                           c["W"], c["sinks"])
    return _prefix(st["q"], st["kp"], st["vp"], st["k"], st["v"], st["len"])


def _angles(st):
    """cos and sin [B, 1, S, R/2] of position * frequency."""
    a = st["pos"].to(F64)[:, None, :, None] * st["inv_freq"].to(F64)
    return torch.cos(a).to(F32), torch.sin(a).to(F32)


def _rotate(y, cos, sin, interleaved):
    """The first R columns of y as R/2 pairs, each turned by its angle."""
    half = cos.shape[-1]
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, y[..., 2 * half:]), dim=-1)


def _norm_rope(x, w, cos, sin, interleaved):
    x = x.to(F32)
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    return _rotate(x * r * w.to(F32), cos, sin, interleaved).to(BF16)


def _norm_rope_bwd(gy, x, w, cos, sin, interleaved):
    x, w = x.to(F32), w.to(F32)
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    g = _rotate(gy.to(F32), cos, -sin, interleaved)  # the rotation's transpose
    xh = x * r
    dw = (g * xh).sum(dim=(0, 1, 2), dtype=F64).to(F32)
    gw = g * w
    dx = r * (gw - xh * (gw * xh).mean(dim=-1, keepdim=True))
    return dx.to(BF16), dw


def _softmax(s):
    """Softmax over the last axis, and the log of its sum; a row of nothing but -inf gives zeros."""
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == NEG, torch.zeros_like(m), m))
    t = p.sum(dim=-1, keepdim=True)
    return p / t.clamp_min(1e-30), m + torch.log(t)


def _scores(q, k, lens, W, sinks):
    """The scaled scores [B, Hkv, group * Sq, Skv], -inf where a query does not see a key."""
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    s = q.to(F32).reshape(B, Hkv, Hq // Hkv * Sq, D) @ k.to(F32).transpose(-1, -2)
    s = (s / math.sqrt(D)).reshape(B, Hkv, Hq // Hkv, Sq, Skv)
    i = lens.long()[:, None] - Sq + torch.arange(Sq, device=q.device)  # the queries' positions
    j = torch.arange(Skv, device=q.device)
    seen = (j <= i[..., None]) & ((i[..., None] - j < W) | (j < sinks))
    return s.masked_fill(~seen[:, None, None], NEG).reshape(B, Hkv, Hq // Hkv * Sq, Skv)


def _window(q, k, v, lens, W, sinks):
    p, lse = _softmax(_scores(q, k, lens, W, sinks))
    return (p @ v.to(F32)).reshape(q.shape).to(BF16), lse.reshape(q.shape[:3])


def _window_bwd(do, q, k, v, o, lse, lens, W, sinks):
    B, Hkv, D = q.shape[0], k.shape[1], q.shape[3]
    s = _scores(q, k, lens, W, sinks)
    p = torch.exp(s - lse.reshape(B, Hkv, -1, 1).clamp_min(-1e30))
    do, o, qf = (t.to(F32).reshape(B, Hkv, -1, D) for t in (do, o, q))
    ds = p * (do @ v.to(F32).transpose(-1, -2) - (do * o).sum(dim=-1, keepdim=True))
    ds = ds / math.sqrt(D)
    dq = (ds @ k.to(F32)).reshape(q.shape)
    dk, dv = ds.transpose(-1, -2) @ qf, p.transpose(-1, -2) @ do
    return dq.to(BF16), dk.to(BF16), dv.to(BF16)


def _prefix(q, kp, vp, k, v, lens):
    B, Hq, Sq, D = q.shape
    Hkv, P, S, rows = kp.shape[0], kp.shape[1], k.shape[2], Hq // kp.shape[0] * Sq
    qf = q.to(F32).reshape(B, Hkv, rows, D)
    shared = qf.transpose(0, 1).reshape(Hkv, B * rows, D) @ kp.to(F32).transpose(-1, -2)
    shared = shared.reshape(Hkv, B, rows, P).transpose(0, 1)
    own_s = qf @ k.to(F32).transpose(-1, -2)
    i = lens.long()[:, None] - Sq + torch.arange(Sq, device=q.device)
    seen = torch.arange(S, device=q.device) <= i[..., None]
    own_s = own_s.reshape(B, Hkv, Hq // Hkv, Sq, S).masked_fill(~seen[:, None, None], NEG)
    p, _ = _softmax(torch.cat((shared, own_s.reshape(B, Hkv, rows, S)), dim=-1) / math.sqrt(D))
    pp = p[..., :P].transpose(0, 1).reshape(Hkv, B * rows, P) @ vp.to(F32)
    o = pp.reshape(Hkv, B, rows, D).transpose(0, 1) + p[..., P:] @ v.to(F32)
    return o.reshape(B, Hq, Sq, D).to(BF16)


# ---------------------------------------------------------------------------
# Work and the definition in 64 bits
# ---------------------------------------------------------------------------
def _seen(n, Sq, W, sinks):
    """Keys that a window call's queries see, over all of them, and in all."""
    pairs, first = 0, n - Sq
    for i in range(max(first, 0), n):
        lo = max(0, i - W + 1)
        pairs += i + 1 - lo + min(sinks, lo)
    lo = max(0, max(first, 0) - W + 1)
    return pairs, (n - lo + min(sinks, lo)) if n > 0 else 0


def work(case):
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    if case["op"] in ("norm_rope", "norm_rope_bwd"):
        n = B * case["S"] * (Hq + Hkv) * D
        small = 4 * B * case["S"] + case["R"] * 2 + 2 * D * case["wbits"] // 8
        if case["op"] == "norm_rope":
            return {"bytes": 4 * n + small, "flops": 8 * n}
        return {"bytes": 6 * n + small + 8 * D, "flops": 16 * n}
    Sq = case["Sq"]
    if case["op"] in ("window", "window_bwd"):
        n = case["Skv"] if case["lens"] == "full" else (max(1, case["Skv"] // 2) + case["Skv"]) // 2
        pairs, keys = _seen(n, Sq, case["W"], case["sinks"])
        if case["op"] == "window_bwd":  # q, o, do, dq; k, v, dk, dv; the row sums
            return {"bytes": 8 * B * Hq * Sq * D + 4 * B * Hkv * (keys + case["Skv"]) * D
                    + 4 * B * Hq * Sq + 4 * B, "flops": 10 * B * Hq * pairs * D}
        return {"bytes": 4 * B * Hq * Sq * D + 4 * B * Hkv * keys * D + 4 * B,
                "flops": 4 * B * Hq * pairs * D}
    n = case["S"] if case["lens"] == "full" else (min(Sq, case["S"]) + case["S"]) // 2
    pairs = Sq * case["P"] + _seen(n, Sq, 1 << 30, 0)[0]
    return {"bytes": 4 * B * Hq * Sq * D + 4 * Hkv * (case["P"] + B * n) * D + 4 * B,
            "flops": 4 * B * Hq * pairs * D}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("norm_rope", "norm_rope_bwd"):
        back = case["op"] == "norm_rope_bwd"
        outs, grads, wgrads = [], [], []
        theta = st["pos"].double().unsqueeze(-1) * st["inv_freq"].double()
        turn = torch.polar(torch.ones_like(theta), theta).unsqueeze(1)
        for x, w, gy in ((st["q"], st["wq"], st.get("gq")), (st["k"], st["wk"], st.get("gk"))):
            w = w.double().requires_grad_(back)
            dw = torch.zeros_like(w)
            dxs, ys = [], []
            for b in range(x.shape[0]):
                xb = x[b:b + 1].double().requires_grad_(back)
                norm = torch.linalg.vector_norm(xb, dim=-1, keepdim=True)
                y = xb / torch.sqrt(norm ** 2 / x.shape[-1] + EPS) * w
                R = case["R"]
                z = y[..., :R].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
                z = z if case["interleaved"] else z.transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[b:b + 1])
                z = z if case["interleaved"] else z.transpose(-1, -2)
                y = torch.cat((z.flatten(-2), y[..., R:]), dim=-1)
                if back:
                    gx, gw = torch.autograd.grad(y, (xb, w), gy[b:b + 1].double())
                    dxs.append(gx)
                    dw = dw + gw
                else:
                    ys.append(y)
            outs.append(torch.cat(ys) if ys else None)
            grads.append(torch.cat(dxs) if dxs else None)
            wgrads.append(dw.detach())
        return (*grads, *wgrads) if back else tuple(outs)
    q, k, v = st["q"], st["k"], st["v"]
    B, Hq, Sq, D = q.shape
    group, lens = Hq // k.shape[1], st["len"].tolist()
    back = case["op"] == "window_bwd"
    out = torch.zeros((B, Hq, Sq, D), dtype=F64, device="cuda")  # o, or dq
    dk, dv = (torch.zeros(k.shape, dtype=F64, device="cuda") if back else None for _ in range(2))
    for b in range(B):
        n = lens[b]
        t = torch.arange(n - Sq, n, device="cuda").unsqueeze(1)
        j = torch.arange(n, device="cuda").unsqueeze(0)
        hide = j > t
        if case["op"] != "prefix":
            hide = hide | ((t - j >= case["W"]) & (j >= case["sinks"]))
        for h in range(k.shape[1]):
            heads = slice(h * group, (h + 1) * group)
            qh, kh, vh = q[b, heads].double(), k[b, h, :n].double(), v[b, h, :n].double()
            mask = hide
            if case["op"] == "prefix":
                kh = torch.cat((st["kp"][h].double(), kh))
                vh = torch.cat((st["vp"][h].double(), vh))
                mask = torch.cat((hide.new_zeros(Sq, case["P"]), hide), dim=1)
            leaves = [x.requires_grad_(back) for x in (qh, kh, vh)]
            s = torch.einsum("gsd,nd->gsn", qh * D ** -0.5, kh).masked_fill(mask, NEG)
            dead = mask.all(dim=-1, keepdim=True)
            o = torch.softmax(s.masked_fill(dead, 0.0), dim=-1).masked_fill(dead, 0.0) @ vh
            if back:
                out[b, heads], dk[b, h, :n], dv[b, h, :n] = torch.autograd.grad(
                    o, leaves, st["do"][b, heads].double())
            else:
                out[b, heads] = o
    return (out, dk, dv) if back else out

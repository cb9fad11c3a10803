"""Plain 64-bit forms of the attention layer's operators, with the error bounds that
their kernels' roundings give.

A bf16 rounding is off by at most 2^-8 of the value; fp32 sums of n terms by at most
n 2^-24 of the sum of the terms' sizes.
"""
from __future__ import annotations

import math

import torch

F64 = torch.float64
BF16_STEP = 2.0 ** -8


def rope_angles(positions, inv_freq, B):
    """positions * inv_freq, [B, 1, S, R/2]."""
    pos = positions if positions.dim() == 2 else positions.unsqueeze(0).expand(B, -1)
    return (pos.to(F64).unsqueeze(-1) * inv_freq.to(F64)).unsqueeze(1)


def rotate(y, angles, interleaved):
    half = angles.shape[-1]
    y = y.clone()
    if interleaved:
        ia, ib = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    else:
        ia, ib = slice(0, half), slice(half, 2 * half)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia] = a * angles.cos() - b * angles.sin()
    y[..., ib] = b * angles.cos() + a * angles.sin()
    return y


def norm_rope(x, w, angles, eps, interleaved):
    """(y, bound of |kernel - y|)."""
    x, w = x.to(F64), w.to(F64)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r * w
    y = rotate(u, angles, interleaved)
    # One bf16 rounding; in fp32 a mean of D squares, rsqrt, three products and an angle's
    # cosine and sine: well under 2^-18 of the row's largest value.
    return y, BF16_STEP * y.abs() + 2.0 ** -18 * u.abs().amax(-1, keepdim=True)


def norm_rope_bwd(gy, x, w, angles, eps, interleaved):
    """(dx, its bound, dw, its bound)."""
    x, w = x.to(F64), w.to(F64)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    g = rotate(gy.to(F64), -angles, interleaved)
    xh = x * r
    gw = g * w
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    size = r * (gw.abs().amax(-1, keepdim=True)
                + xh.abs().amax(-1, keepdim=True) * (gw * xh).abs().mean(-1, keepdim=True))
    dw = (g * xh).sum((0, 1, 2))
    # fp32 sums of at most a few hundred terms, three levels deep: 2^-16 of the terms' sizes.
    # (g is a turned pair: its own error is 2^-20 of the pair, covered by the row maximum.)
    dw_size = (g.abs().amax(-1, keepdim=True) * xh.abs()).sum((0, 1, 2))
    return dx, BF16_STEP * dx.abs() + 2.0 ** -17 * size, dw, 2.0 ** -16 * dw_size


def visible(lens, Sq, Skv, window, sinks, device):
    """[B, 1, Sq, Skv]: query i of request b, at lens[b] - Sq + i, sees key j."""
    i = lens.to(torch.int64)[:, None, None] - Sq + torch.arange(Sq, device=device)[None, :, None]
    j = torch.arange(Skv, device=device)[None, None, :]
    return ((j <= i) & ((i - j < window) | (j < sinks))).unsqueeze(1)


def _heads(t, group):
    return t.to(F64).repeat_interleave(group, dim=1)


def _masked(t, rows):
    """t with the rows that nothing sees, or that see nothing, replaced by zeros."""
    return torch.where(rows, t.to(F64), torch.zeros((), dtype=F64, device=t.device))


def attention(q, k, v, seen, scale=-1.0):
    """(o, bound, lse, bound) over the keys that `seen` [B, 1, Sq, Skv] leaves."""
    D, group = q.shape[-1], q.shape[1] // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale < 0 else scale
    used = seen.any(2).unsqueeze(-1)                      # [B, 1, Skv, 1]
    k, v = _masked(k, used), _masked(v, used)
    q = _masked(q, seen.any(-1, keepdim=True))
    kh, vh = _heads(k, group), _heads(v, group)
    s = (q @ kh.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)), 0.0)
    o = p @ vh
    # Scores: fp32 sums of D products, off by D 2^-24 of their sizes; each weight then by that
    # and by 2^-13 (exp2 on the FMA pipe at D = 64, 7.5e-5), and by the bf16 rounding with
    # which it enters the second product.
    e_s = (q.abs() @ kh.abs().transpose(-1, -2)).amax() * scale * D * 2.0 ** -24
    rel = BF16_STEP + 2.0 ** -13 + 2 * e_s
    bound = BF16_STEP * o.abs() + rel * (p @ vh.abs()) + 1e-30
    return o, bound, lse.squeeze(-1), e_s + 2.0 ** -13 + 2.0 ** -20 * lse.abs().squeeze(-1)


def attention_bwd(dout, q, k, v, o, lse, seen, scale=-1.0):
    """((dq, bound), (dk, bound), (dv, bound)) from the given o and lse."""
    B, Hq, Sq, D = q.shape
    Hkv, group = k.shape[1], Hq // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale < 0 else scale
    used, sees = seen.any(2).unsqueeze(-1), seen.any(-1, keepdim=True)
    k, v = _masked(k, used), _masked(v, used)
    q, dout, o = _masked(q, sees), _masked(dout, sees), _masked(o, sees)
    kh, vh = _heads(k, group), _heads(v, group)
    s = q @ kh.transpose(-1, -2) * scale
    row = torch.where(torch.isinf(lse), 0.0, lse.to(F64)).unsqueeze(-1)
    p = torch.where(seen, torch.exp(s - row), 0.0)
    dp = dout @ vh.transpose(-1, -2)
    ds = p * (dp - (dout * o).sum(-1, keepdim=True))

    def shared(t):
        return t.reshape(B, Hkv, group, -1, D).sum(2)

    dq = ds @ kh * scale
    dk = shared(ds.transpose(-1, -2) @ q) * scale
    dv = shared(p.transpose(-1, -2) @ dout)
    # The weights' own error (scores as above, lse given in fp32) and the fp32 error of
    # dp - delta, 2 D 2^-24 of its terms; p and ds enter the last products in bf16.
    e_s = ((q.abs() @ kh.abs().transpose(-1, -2)).amax() * scale * D
           + lse.to(F64).abs().masked_fill(torch.isinf(lse), 0.0).amax()) * 2.0 ** -24
    e_dp = ((dout.abs() @ vh.abs().transpose(-1, -2)).amax()
            + (dout * o).abs().sum(-1).amax()) * 2 * D * 2.0 ** -24
    rel = BF16_STEP + 2.0 ** -13 + 2 * e_s
    e_ds = rel * ds.abs() + e_dp * p
    return ((dq, BF16_STEP * dq.abs() + e_ds @ kh.abs() * scale + 1e-30),
            (dk, BF16_STEP * dk.abs() + shared(e_ds.transpose(-1, -2) @ q.abs()) * scale + 1e-30),
            (dv, BF16_STEP * dv.abs() + shared(rel * p.transpose(-1, -2) @ dout.abs()) + 1e-30))


def shared_prefix(q, kp, vp, k, v, lens, scale=-1.0):
    """(o, bound): the prefix keys before each request's own."""
    B, P = q.shape[0], kp.shape[1]
    own = visible(lens, q.shape[2], k.shape[2], 1 << 40, 0, q.device)
    seen = torch.cat((own.new_ones(*own.shape[:3], P), own), dim=-1)
    full = [torch.cat((p.unsqueeze(0).expand(B, -1, -1, -1), t), dim=2)
            for p, t in ((kp, k), (vp, v))]
    return attention(q, *full, seen, scale)[:2]


def check_close(got, want, bound, what=""):
    got = got.to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs() - bound
    assert off.max().item() <= 0, (
        f"{what}: off by {(got - want).abs().max().item():.3e}, "
        f"{off.max().item():.3e} past the bound")

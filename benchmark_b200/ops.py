"""torch-tensor conveniences over the C ABI.

Tensors are bf16, contiguous, on the current CUDA device; the calls run on the
current torch stream.  torch is only the device-memory and stream plumbing:
all arithmetic happens in libb200attn.so's CUDA kernels.

The attention layer's operators (qk_norm_rope, attention_window_*,
attention_shared_prefix) take [B, H, S, D] views of any strides with D
contiguous, on any one device; they run on that device's current stream or on
`stream`, where their outputs and workspaces are allocated too.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib


def _stream_ptr(stream: torch.cuda.Stream | None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _check_bf16(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("expected contiguous bf16 CUDA tensors")


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  out: torch.Tensor | None = None, causal: bool = False,
                  softmax_scale: float = -1.0, stream: torch.cuda.Stream | None = None,
                  scalar: bool = False) -> torch.Tensor:
    """q [B,Hq,Sq,D], k/v [B,Hkv,Skv,D] -> o [B,Hq,Sq,D] (bf16).

    scalar=True runs the validation-only CUDA-core kernel instead of the fused one."""
    _check_bf16(q, k, v)
    B, Hq, Sq, D = q.shape
    Bk, Hkv, Skv, Dk = k.shape
    if Bk != B or Dk != D or tuple(v.shape) != tuple(k.shape):
        raise ValueError("q/k/v shapes disagree")
    if out is None:
        out = torch.empty_like(q)
    _check_bf16(out)
    name = "attention_fwd_scalar" if scalar else "attention_fwd"
    _lib.call(name, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, Hq, Hkv, Sq,
              Skv, D, int(bool(causal)), float(softmax_scale), _stream_ptr(stream))
    return out


def fill_normal_(t: torch.Tensor, seed: int, tensor_id: int, mean: float = 0.0,
                 sigma: float = 1.0, index_base: int = 0,
                 stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    _check_bf16(t)
    _lib.call("b200_fill_normal_bf16", t.data_ptr(), t.numel(), seed, tensor_id, index_base,
              mean, sigma, _stream_ptr(stream))
    return t


def fill_uniform_(t: torch.Tensor, seed: int, tensor_id: int, lo: float = -1.0, hi: float = 1.0,
                  index_base: int = 0, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    _check_bf16(t)
    _lib.call("b200_fill_uniform_bf16", t.data_ptr(), t.numel(), seed, tensor_id, index_base,
              lo, hi, _stream_ptr(stream))
    return t


def check(stream: torch.cuda.Stream | None = None) -> None:
    """Synchronise and raise B200Error(B200_ETIMEOUT) if a device wait gave up."""
    _lib.call("b200_check", _stream_ptr(stream))


def gemm_bf16(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None,
              b_col_major: bool = True, impl: str = "tcgen05",
              stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """C [M,N] (bf16) = A [M,K] @ B, B given as [N,K] (b_col_major) or [K,N].

    impl: "tcgen05" (this library's kernel) or "cublas" (comparator)."""
    _check_bf16(a, b)
    M, K = a.shape
    N = b.shape[0] if b_col_major else b.shape[1]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=a.device)
    name = {"tcgen05": "gemm_bf16", "cublas": "gemm_bf16_cublas"}[impl]
    _lib.call(name, a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, int(b_col_major),
              _stream_ptr(stream))
    return out


def gemm_f32_reference(a: torch.Tensor, b: torch.Tensor, b_col_major: bool = True,
                       stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    _check_bf16(a, b)
    M, K = a.shape
    N = b.shape[0] if b_col_major else b.shape[1]
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    _lib.call("gemm_f32_reference", a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K,
              int(b_col_major), _stream_ptr(stream))
    return out


# ---------------------------------------------------------------------------
# Operators of the attention layer
# ---------------------------------------------------------------------------
def _on_its_device(fn):
    """Run fn with its first tensor's device current and `stream`, if given, as the
    current stream, so that what it allocates belongs to that stream."""
    @functools.wraps(fn)
    def call(first, *args, stream: torch.cuda.Stream | None = None, **kwargs):
        if not first.is_cuda:
            raise ValueError("expected CUDA tensors")
        if stream is not None:
            if stream.device != first.device:
                raise ValueError("stream and tensors are on different devices")
            with torch.cuda.stream(stream):
                return fn(first, *args, **kwargs)
        if first.device.index != torch.cuda.current_device():
            with torch.cuda.device(first.device):
                return fn(first, *args, **kwargs)
        return fn(first, *args, **kwargs)
    return call


def _view(t: torch.Tensor, shape: tuple, device: torch.device, name: str) -> _lib.Tensor:
    if t.dtype != torch.bfloat16 or t.device != device:
        raise ValueError(f"{name}: expected a bf16 tensor on {device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
    sb, sh, ss, sd = t.stride()
    if sd != 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    return _lib.Tensor(t.data_ptr(), sb, sh, ss)


def _flat_ptr(t: torch.Tensor | None, dtype: torch.dtype, shape: tuple, device: torch.device,
              name: str) -> int | None:
    if t is None:
        return None
    if t.dtype != dtype or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {shape} on {device}")
    return t.data_ptr()


def _empty(shape, device, dtype=torch.bfloat16) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=device)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name: str, device: int, *args: int) -> int:
    """What the named entry point needs for these sizes on this (current) device."""
    n = ctypes.c_size_t()
    _lib.call(name, *args, ctypes.byref(n))
    return n.value


def _workspace(name: str, device: torch.device, *args: int) -> tuple[torch.Tensor | None, int, int]:
    n = _workspace_bytes(name, device.index, *args)
    if n == 0:
        return None, 0, 0
    w = _empty(n, device, torch.uint8)
    return w, w.data_ptr(), n


def _rope_args(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved):
    B, Hq, S, D = q.shape
    Hkv = k.shape[1]
    dev = q.device
    wt = torch.float32 if q_weight.dtype == torch.float32 else torch.bfloat16
    wq = _flat_ptr(q_weight, wt, (D,), dev, "q_weight")
    wk = _flat_ptr(k_weight, wt, (D,), dev, "k_weight")
    f = _flat_ptr(inv_freq, torch.float32, (inv_freq.numel(),), dev, "inv_freq")
    if (positions.dtype != torch.int32 or positions.device != dev
            or tuple(positions.shape) not in ((S,), (B, S))
            or (S > 1 and positions.stride(-1) != 1)):
        raise ValueError(f"positions: expected int32 [{S}] or [{B}, {S}] on {dev}, "
                         "contiguous along the tokens")
    pos_sb = positions.stride(0) if positions.dim() == 2 and B > 1 else 0
    return (_view(q, (B, Hq, S, D), dev, "q"), _view(k, (B, Hkv, S, D), dev, "k"), wq, wk,
            int(wt == torch.float32), f, 2 * inv_freq.numel(), int(bool(interleaved)),
            positions.data_ptr(), pos_sb, float(eps))


@_on_its_device
def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor,
                 eps: float = 1e-6, interleaved: bool = False,
                 q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm of each query and key head with the rotation by position, in one pass.

    q [B,Hq,S,D], k [B,Hkv,S,D] (any strides, D contiguous; D 64 or 128);
    q_weight, k_weight [D] bf16 or fp32; inv_freq [R/2] fp32: the first R columns (a
    multiple of 16, at most D) turn by position * inv_freq, in halves or as adjacent
    pairs (interleaved); positions int32 [B,S] or [S].  q_out and k_out default to
    contiguous [B,H,S,D]; they may be q and k themselves, or a cache's rows."""
    B, Hq, S, D = q.shape
    Hkv, dev = k.shape[1], q.device
    args = _rope_args(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved)
    if q_out is None:
        q_out = _empty((B, Hq, S, D), dev)
    if k_out is None:
        k_out = _empty((B, Hkv, S, D), dev)
    _lib.call("qk_norm_rope", *args, _view(q_out, (B, Hq, S, D), dev, "q_out"),
              _view(k_out, (B, Hkv, S, D), dev, "k_out"), B, S, Hq, Hkv, D, _stream_ptr(None))
    return q_out, k_out


@_on_its_device
def qk_norm_rope_bwd(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor,
                     k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                     inv_freq: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                     interleaved: bool = False, dq: torch.Tensor | None = None,
                     dk: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """Gradients of qk_norm_rope: (dq, dk, dq_weight, dk_weight), the last two fp32 [D].

    dq_out, dk_out: the gradients of its outputs; the rest are its inputs.  dq and dk
    default to contiguous [B,H,S,D]; they may be dq_out and dk_out themselves."""
    B, Hq, S, D = q.shape
    Hkv, dev = k.shape[1], q.device
    args = _rope_args(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved)
    gq = _view(dq_out, (B, Hq, S, D), dev, "dq_out")
    gk = _view(dk_out, (B, Hkv, S, D), dev, "dk_out")
    if dq is None:
        dq = _empty((B, Hq, S, D), dev)
    if dk is None:
        dk = _empty((B, Hkv, S, D), dev)
    dw = _empty((2, D), dev, torch.float32)
    w, w_ptr, w_bytes = _workspace("qk_norm_rope_bwd_workspace", dev, B, S, D)
    _lib.call("qk_norm_rope_bwd", gq, gk, *args, _view(dq, (B, Hq, S, D), dev, "dq"),
              _view(dk, (B, Hkv, S, D), dev, "dk"), dw.data_ptr(), dw.data_ptr() + 4 * D, B, S,
              Hq, Hkv, D, w_ptr, w_bytes, _stream_ptr(None))
    return dq, dk, dw[0], dw[1]


@_on_its_device
def attention_window_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                         sinks: int = 0, kv_len: torch.Tensor | None = None,
                         out: torch.Tensor | None = None, softmax_scale: float = -1.0,
                         lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention with a sliding window and sink tokens: q [B,Hq,Sq,D], k/v [B,Hkv,Skv,D]
    (any strides, D contiguous) -> o [B,Hq,Sq,D].

    Request b has kv_len[b] keys (int32 [B]; default Skv) and its queries are the last Sq
    positions; the query at position p sees key j iff j <= p and (p - j < window or
    j < sinks).  A query that sees nothing gives zeros.  lse, if given (fp32 [B,Hq,Sq]),
    receives the rows' log-sum-exp, which attention_window_bwd reads."""
    B, Hq, Sq, D = q.shape
    _, Hkv, Skv, _ = k.shape
    dev = q.device
    if out is None:
        out = _empty((B, Hq, Sq, D), dev)
    window, sinks = min(int(window), 0x7fffffff), min(int(sinks), 0x7fffffff)
    tensors = (_view(q, (B, Hq, Sq, D), dev, "q"), _view(k, (B, Hkv, Skv, D), dev, "k"),
               _view(v, (B, Hkv, Skv, D), dev, "v"), _view(out, (B, Hq, Sq, D), dev, "out"))
    lse_ptr = _flat_ptr(lse, torch.float32, (B, Hq, Sq), dev, "lse")
    len_ptr = _flat_ptr(kv_len, torch.int32, (B,), dev, "kv_len")
    w, w_ptr, w_bytes = _workspace("attention_window_fwd_workspace", dev, B, Hq, Hkv, Sq, Skv, D,
                                   window, sinks)
    _lib.call("attention_window_fwd", *tensors, lse_ptr, len_ptr, B, Hq, Hkv, Sq, Skv, D, window,
              sinks, float(softmax_scale), w_ptr, w_bytes, _stream_ptr(None))
    return out


@_on_its_device
def attention_window_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         o: torch.Tensor, lse: torch.Tensor, window: int, sinks: int = 0,
                         kv_len: torch.Tensor | None = None, softmax_scale: float = -1.0,
                         dq: torch.Tensor | None = None, dk: torch.Tensor | None = None,
                         dv: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """Gradients of attention_window_fwd: (dq, dk, dv).

    dout: the gradient of o; o and lse: what the forward call wrote; the rest are its
    arguments.  dq, dk and dv default to contiguous tensors."""
    B, Hq, Sq, D = q.shape
    _, Hkv, Skv, _ = k.shape
    dev = q.device
    qs, ks = (B, Hq, Sq, D), (B, Hkv, Skv, D)
    dq = _empty(qs, dev) if dq is None else dq
    dk = _empty(ks, dev) if dk is None else dk
    dv = _empty(ks, dev) if dv is None else dv
    window, sinks = min(int(window), 0x7fffffff), min(int(sinks), 0x7fffffff)
    ins = (_view(dout, qs, dev, "dout"), _view(q, qs, dev, "q"), _view(k, ks, dev, "k"),
           _view(v, ks, dev, "v"), _view(o, qs, dev, "o"))
    outs = (_view(dq, qs, dev, "dq"), _view(dk, ks, dev, "dk"), _view(dv, ks, dev, "dv"))
    lse_ptr = _flat_ptr(lse, torch.float32, (B, Hq, Sq), dev, "lse")
    len_ptr = _flat_ptr(kv_len, torch.int32, (B,), dev, "kv_len")
    w, w_ptr, w_bytes = _workspace("attention_window_bwd_workspace", dev, B, Hq, Sq)
    _lib.call("attention_window_bwd", *ins, lse_ptr, *outs, len_ptr, B, Hq, Hkv, Sq, Skv, D,
              window, sinks, float(softmax_scale), w_ptr, w_bytes, _stream_ptr(None))
    return dq, dk, dv


@_on_its_device
def attention_shared_prefix(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                            k: torch.Tensor, v: torch.Tensor, kv_len: torch.Tensor | None = None,
                            out: torch.Tensor | None = None,
                            softmax_scale: float = -1.0) -> torch.Tensor:
    """Attention of a batch behind a prefix that all its requests share.

    q [B,Hq,Sq,D]; k_prefix/v_prefix [Hkv,P,D]; k/v [B,Hkv,S,D]: each request's own keys
    (any strides, D contiguous) -> o [B,Hq,Sq,D].  Query i of request b sees the whole
    prefix and its own keys j <= kv_len[b] - Sq + i (int32 [B]; default S)."""
    B, Hq, Sq, D = q.shape
    Hkv, P, _ = k_prefix.shape
    S, dev = k.shape[2], q.device
    if out is None:
        out = _empty((B, Hq, Sq, D), dev)
    kv_p = (1, Hkv, P, D)
    tensors = (_view(q, (B, Hq, Sq, D), dev, "q"),
               _view(k_prefix.unsqueeze(0), kv_p, dev, "k_prefix"),
               _view(v_prefix.unsqueeze(0), kv_p, dev, "v_prefix"),
               _view(k, (B, Hkv, S, D), dev, "k"), _view(v, (B, Hkv, S, D), dev, "v"),
               _view(out, (B, Hq, Sq, D), dev, "out"))
    len_ptr = _flat_ptr(kv_len, torch.int32, (B,), dev, "kv_len")
    w, w_ptr, w_bytes = _workspace("attention_shared_prefix_workspace", dev, B, Hq, Hkv, Sq, P, S,
                                   D)
    _lib.call("attention_shared_prefix", *tensors, len_ptr, B, Hq, Hkv, Sq, P, S, D,
              float(softmax_scale), w_ptr, w_bytes, _stream_ptr(None))
    return out

"""torch-tensor conveniences over the C ABI.

Tensors are bf16, contiguous, on the current CUDA device; the calls run on the
current torch stream.  torch is only the device-memory and stream plumbing:
all arithmetic happens in libb200attn.so's CUDA kernels.

The attention layer's operators (qk_norm_rope, attention_window_*,
attention_shared_prefix) take [B, H, S, D] views of any strides with D
contiguous, on any one device; they run on that device's current stream or on
`stream`, where their outputs and workspaces are allocated too.

No call records a gradient: outputs have no history, whatever their inputs require.
The `_bwd` functions are for a torch.autograd.Function of the caller's.
"""
from __future__ import annotations

import importlib

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
_binding = None


def binding():
    """The torch extension that these operators' calls go through (csrc/binding.cpp)."""
    global _binding
    if _binding is None:
        _lib.lib()
        try:
            _binding = importlib.import_module("benchmark_b200._binding")
        except ModuleNotFoundError as e:
            raise ImportError("benchmark_b200/_binding.so is not built; run `python -m "
                              "benchmark_b200.build` (there is no fallback)") from e
    return _binding


def _call(name: str, stream: torch.cuda.Stream | None, *args):
    fn = getattr(_binding or binding(), name)
    if stream is None:
        return fn(*args)
    device = getattr(args[0], "device", None)
    if device != stream.device:
        raise ValueError(f"{name}: the stream is on {stream.device}, the tensors on {device}")
    with torch.cuda.stream(stream):  # what the call allocates belongs to that stream
        return fn(*args)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor,
                 eps: float = 1e-6, interleaved: bool = False,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm of each query and key head with the rotation by position, in one pass.

    q [B,Hq,S,D], k [B,Hkv,S,D] (any strides, D contiguous; D 64 or 128);
    q_weight, k_weight [D] bf16 or fp32; inv_freq [R/2] fp32: the first R columns (a
    multiple of 16, at most D) turn by position * inv_freq, in halves or as adjacent
    pairs (interleaved); positions int32 [B,S] or [S].  q_out and k_out default to
    contiguous [B,H,S,D]; they may be q and k themselves, or a cache's rows."""
    return _call("qk_norm_rope", stream, q, k, q_weight, k_weight, inv_freq, positions, eps,
                 interleaved, q_out, k_out)


def qk_norm_rope_bwd(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor,
                     k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                     inv_freq: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                     interleaved: bool = False, dq: torch.Tensor | None = None,
                     dk: torch.Tensor | None = None,
                     stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, ...]:
    """Gradients of qk_norm_rope: (dq, dk, dq_weight, dk_weight), the last two fp32 [D].

    dq_out, dk_out: the gradients of its outputs; the rest are its inputs.  dq and dk
    default to contiguous [B,H,S,D]; they may be dq_out and dk_out themselves."""
    return _call("qk_norm_rope_bwd", stream, dq_out, dk_out, q, k, q_weight, k_weight, inv_freq,
                 positions, eps, interleaved, dq, dk)


def attention_window_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                         sinks: int = 0, kv_len: torch.Tensor | None = None,
                         out: torch.Tensor | None = None, softmax_scale: float = -1.0,
                         lse: torch.Tensor | None = None,
                         stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention with a sliding window and sink tokens: q [B,Hq,Sq,D], k/v [B,Hkv,Skv,D]
    (any strides, D contiguous) -> o [B,Hq,Sq,D].

    Request b has kv_len[b] keys (int32 [B]; default Skv) and its queries are the last Sq
    positions; the query at position p sees key j iff j <= p and (p - j < window or
    j < sinks).  A query that sees nothing gives zeros.  lse, if given (fp32 [B,Hq,Sq]),
    receives the rows' log-sum-exp, which attention_window_bwd reads."""
    return _call("attention_window_fwd", stream, q, k, v, window, sinks, kv_len, out,
                 softmax_scale, lse)


def attention_window_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         o: torch.Tensor, lse: torch.Tensor, window: int, sinks: int = 0,
                         kv_len: torch.Tensor | None = None, softmax_scale: float = -1.0,
                         dq: torch.Tensor | None = None, dk: torch.Tensor | None = None,
                         dv: torch.Tensor | None = None,
                         stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, ...]:
    """Gradients of attention_window_fwd: (dq, dk, dv).

    dout: the gradient of o; o and lse: what the forward call wrote; the rest are its
    arguments.  dq, dk and dv default to contiguous tensors."""
    return _call("attention_window_bwd", stream, dout, q, k, v, o, lse, window, sinks, kv_len,
                 softmax_scale, dq, dk, dv)


def attention_shared_prefix(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                            k: torch.Tensor, v: torch.Tensor, kv_len: torch.Tensor | None = None,
                            out: torch.Tensor | None = None, softmax_scale: float = -1.0,
                            stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention of a batch behind a prefix that all its requests share.

    q [B,Hq,Sq,D]; k_prefix/v_prefix [Hkv,P,D]; k/v [B,Hkv,S,D]: each request's own keys
    (any strides, D contiguous) -> o [B,Hq,Sq,D].  Query i of request b sees the whole
    prefix and its own keys j <= kv_len[b] - Sq + i (int32 [B]; default S).

    Made for decoding: with Hq / Hkv * Sq above 128 (a prompt) a request reads the prefix
    again for every 16 of these rows, and attention_window_fwd over caches that hold a copy
    of the prefix is faster."""
    return _call("attention_shared_prefix", stream, q, k_prefix, v_prefix, k, v, kv_len, out,
                 softmax_scale)

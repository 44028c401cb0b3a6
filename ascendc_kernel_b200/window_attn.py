"""Attention with a sliding window and a few first tokens that stay visible.

The reference's ``ModelArgs`` declares ``window_size`` (reference/task2_v0_ref.py:21-61)
and holds no attention that uses it; this is that operator next to
:mod:`ascendc_kernel_b200.sparse_attn`, with the same per-head sink logits and with keys
and values that may be one tensor. Prompts and training steps run here
(:func:`window_attn`, differentiable); single new tokens over a paged cache run in
:mod:`ascendc_kernel_b200.paged_cache` under the same mask.

Shape preconditions are checked with ``assert``; CUDA-level failures raise DsaError.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn as nn

from ._native import call

DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # DSA_DTYPE_*


def _strided(x: torch.Tensor) -> torch.Tensor:
    """x itself when the kernels can step over its strides, else a contiguous copy."""
    ok = x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and all(
        n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(x.shape[:-1], x.stride()[:-1]))
    if ok:
        return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _strides(x: torch.Tensor):
    return (ctypes.c_int64 * 3)(*x.stride()[:3])


def _check(q, k, v, sink, window, n_first, kv_lens, softmax_scale):
    assert q.is_cuda and k.is_cuda and (v is None or v.is_cuda), "inputs must be CUDA tensors"
    assert q.dtype in DTYPES, "q must be bf16 or fp16"
    assert q.dim() == 4 and k.dim() == 4, "q is [b, m, h, d], k and v are [b, n, hk, d]"
    b, m, h, d = q.shape
    assert k.dtype == q.dtype and k.device == q.device, "q, k and v have one type and device"
    assert k.shape[0] == b and k.shape[3] == d, "k must be [b, n, hk, d]"
    if v is not None:
        assert v.shape == k.shape and v.dtype == q.dtype and v.device == q.device, \
            "v must be like k"
    hk = k.shape[2]
    assert d in (64, 128), "kernel specialised to head_dim in (64, 128)"
    assert hk >= 1 and h % hk == 0 and 1 <= h // hk <= 128, \
        "n_heads must be a multiple of n_kv_heads, at most 128 to a group"
    assert window >= 1 and n_first >= 0, "window >= 1 and n_first >= 0"
    assert softmax_scale > 0, "softmax_scale must be positive"
    if sink is not None:
        assert sink.numel() == h, "sink must have n_heads entries"
    if kv_lens is not None:
        assert kv_lens.is_cuda and kv_lens.device == q.device and kv_lens.dtype == torch.int32 \
            and kv_lens.shape == (b,), "kv_lens must be int32 [b] on q's device"


def _sink_on(sink, device):
    if sink is None:
        return None
    return sink.detach().to(device=device, dtype=torch.float32).contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


def _forward(q, k, v, sink, window, n_first, kv_lens, scale, out, want_lse):
    """Launches the forward; v None: the keys serve as values. Returns out and lse."""
    b, m, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    q, k = _strided(q), _strided(k)
    v = k if v is None else _strided(v)
    kv_lens = None if kv_lens is None else kv_lens.contiguous()
    if out is None:
        out = torch.empty(b, m, h, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, m, h, dtype=torch.float32, device=q.device) if want_lse else None
    stream = torch.cuda.current_stream(q.device).cuda_stream
    with torch.cuda.device(q.device):
        call("dsa_window_attn_fwd", q.data_ptr(), _strides(q), k.data_ptr(), _strides(k),
             v.data_ptr(), _strides(v), _ptr(sink), _ptr(kv_lens), out.data_ptr(), _ptr(lse),
             DTYPES[q.dtype], b, m, n, h, hk, d, window, n_first, scale, stream)
    return out, lse


def window_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None = None,
                sink: torch.Tensor | None = None, *, window: int, n_first: int = 0,
                kv_lens: torch.Tensor | None = None, softmax_scale: float | None = None,
                out: torch.Tensor | None = None, return_lse: bool = False):
    """out[b,t,h] = sum_j softmax_j(q.k_j * scale ++ sink[h]) v_j over the keys t sees.

    q [b, m, h, d], k and v [b, n, hk, d], bf16 or fp16, d 64 or 128, h a multiple of hk
    (v None: the keys serve as values). Query t stands at position p = t + n - m and sees
    key j when j <= p, j < kv_lens[b] (int32 [b], default n) and j > p - window or
    j < n_first. sink [h] fp32 logits or None; softmax_scale defaults to d ** -0.5. Rows
    that see nothing and have no sink are 0. Returns out like q, and with ``return_lse``
    also the fp32 log of the softmax divisor [b, m, h].

    Differentiable in q, k, v and sink (``out`` must then be None).
    """
    scale = float(q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale)
    _check(q, k, v, sink, window, n_first, kv_lens, scale)
    window, n_first = min(int(window), 1 << 28), min(int(n_first), 1 << 28)
    if out is not None:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device \
            and out.is_contiguous(), "out must be contiguous and like q"
    out, lse = _forward(q, k, v, _sink_on(sink, q.device), window, n_first, kv_lens, scale, out,
                        return_lse)
    return (out, lse) if return_lse else out

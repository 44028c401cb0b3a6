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

from ._native import bind, lib

try:  # the current stream's raw handle without building a Stream object
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # pragma: no cover - older torch
    def _raw_stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream

DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # DSA_DTYPE_*


def _strided(x: torch.Tensor) -> torch.Tensor:
    """x itself when the kernels can step over its strides, else a contiguous copy."""
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x
    ok = x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and all(
        n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(x.shape[:-1], x.stride()[:-1]))
    if ok:
        return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


_I64x3 = ctypes.c_int64 * 3


def _strides(x: torch.Tensor):
    """The first three strides for the C ABI; None (contiguous) where they are that."""
    return None if x.is_contiguous() else _I64x3(*x.stride()[:3])


_entries = {}


def _run(fn: str, dev: int, *args) -> None:
    """Calls entry point `fn` on device `dev` with the current stream there as the last
    argument. The entry points are bound once, and the device guard is entered only for a
    device that is not the current one: the calls are a few microseconds long."""
    entry = _entries.get(fn)
    if entry is None:
        entry = _entries[fn] = bind(fn)
    if dev == torch.cuda.current_device():
        entry(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            entry(*args, _raw_stream(dev))


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
    if sink is None or (sink.dtype == torch.float32 and sink.device == device
                        and sink.is_contiguous()):
        return sink
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
    _run("dsa_window_attn_fwd", q.get_device(), q.data_ptr(), _strides(q), k.data_ptr(),
         _strides(k), v.data_ptr(), _strides(v), _ptr(sink), _ptr(kv_lens), out.data_ptr(),
         _ptr(lse), DTYPES[q.dtype], b, m, n, h, hk, d, window, n_first, scale)
    return out, lse


def window_attn_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                    v: torch.Tensor | None, sink: torch.Tensor | None, out: torch.Tensor,
                    lse: torch.Tensor, *, window: int, n_first: int = 0,
                    kv_lens: torch.Tensor | None = None, softmax_scale: float | None = None):
    """Gradients of :func:`window_attn` from its inputs, its ``out`` and ``lse`` and the
    upstream gradient ``dout``: (dq, dk, dv, dsink), contiguous and of the inputs' types (dv
    None when v is None: dk is then the gradient of the shared tensor; dsink fp32, None
    without a sink). Runs in a fixed order: the same inputs give the same bits."""
    scale = float(q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale)
    _check(q, k, v, sink, window, n_first, kv_lens, scale)
    window, n_first = min(int(window), 1 << 28), min(int(n_first), 1 << 28)
    b, m, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    for x in (dout, out):
        assert x.shape == q.shape and x.dtype == q.dtype and x.device == q.device, \
            "dout and out must be like q"
    assert out.is_contiguous(), "out must be contiguous"
    assert lse.shape == (b, m, h) and lse.dtype == torch.float32 and lse.is_contiguous() \
        and lse.device == q.device, "lse must be fp32 [b, m, h], contiguous"
    q, k, dout = _strided(q), _strided(k), _strided(dout)
    values = k if v is None else _strided(v)
    sink = _sink_on(sink, q.device)
    kv_lens = None if kv_lens is None else kv_lens.contiguous()
    dev = q.device
    dq = torch.empty(b, m, h, d, dtype=q.dtype, device=dev)
    dk = torch.empty(b, n, hk, d, dtype=q.dtype, device=dev)
    dv = None if v is None else torch.empty_like(dk)
    dsink = None if sink is None else torch.empty(h, dtype=torch.float32, device=dev)
    nbytes = lib().dsa_window_attn_bwd_workspace_bytes(b, m, n, h, hk, d, window, n_first,
                                                       1 if v is None else 0)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
    _run("dsa_window_attn_bwd", q.get_device(), q.data_ptr(), _strides(q), k.data_ptr(),
         _strides(k), values.data_ptr(), _strides(values), _ptr(sink), _ptr(kv_lens),
         out.data_ptr(), lse.data_ptr(), dout.data_ptr(), _strides(dout), dq.data_ptr(),
         dk.data_ptr(), _ptr(dv), _ptr(dsink), DTYPES[q.dtype], b, m, n, h, hk, d, window,
         n_first, scale, ws.data_ptr(), ws.numel())
    return dq, dk, dv, dsink


class _WindowAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sink, window, n_first, kv_lens, scale):
        out, lse = _forward(q, k, v, _sink_on(sink, q.device), window, n_first, kv_lens, scale,
                            None, True)
        ctx.save_for_backward(q, k, v, sink, kv_lens, out, lse)
        ctx.args = (window, n_first, scale)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        if dlse is not None:
            raise RuntimeError("the lse of window_attn has no gradient: detach it in the loss")
        if dout is None:
            return (None,) * 8
        q, k, v, sink, kv_lens, out, lse = ctx.saved_tensors
        window, n_first, scale = ctx.args
        dq, dk, dv, dsink = window_attn_bwd(dout, q, k, v, sink, out, lse, window=window,
                                            n_first=n_first, kv_lens=kv_lens,
                                            softmax_scale=scale)
        if dsink is not None:
            dsink = dsink.to(device=sink.device, dtype=sink.dtype).reshape(sink.shape)
        return dq, dk, dv, dsink, None, None, None, None


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

    Positions are the same in every sequence: ``kv_lens`` hides keys and moves no query. It
    is for prompts padded on the right (m = n). The next chunk of sequences whose prefixes
    differ in length has a position of its own in each: give each length a call, with k and
    v cut to it (n = kv_lens[b]).

    The softmax's weights are rounded to q's type before they meet v (its maxima, sums and
    products are fp32), in the backward pass dS too: an error of the size of the results'
    own rounding.

    out is differentiable in q, k, v and sink (the ``out`` argument must then be None). lse is
    not: a backward pass that reaches it raises RuntimeError.
    """
    scale = float(q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale)
    _check(q, k, v, sink, window, n_first, kv_lens, scale)
    window, n_first = min(int(window), 1 << 28), min(int(n_first), 1 << 28)
    if out is not None:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device \
            and out.is_contiguous(), "out must be contiguous and like q"
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, sink)):
        assert out is None, "a differentiable call allocates its own out"
        out, lse = _WindowAttn.apply(q, k, v, sink, window, n_first, kv_lens, scale)
        return (out, lse) if return_lse else out
    out, lse = _forward(q, k, v, _sink_on(sink, q.device), window, n_first, kv_lens, scale, out,
                        return_lse)
    return (out, lse) if return_lse else out


class WindowAttention(nn.Module):
    """:func:`window_attn` with its window and a learned sink logit per head, as
    :class:`ascendc_kernel_b200.sparse_attn.ModelNew` holds them. ``window`` defaults to the
    reference's ``ModelArgs.window_size``."""

    def __init__(self, n_heads: int, head_dim: int, window: int = 128, n_first: int = 0):
        super().__init__()
        self.n_heads = n_heads
        self.head_dim = head_dim
        self.window = window
        self.n_first = n_first
        self.softmax_scale = head_dim ** -0.5
        self.attn_sink = nn.Parameter(torch.zeros(n_heads, dtype=torch.float32))

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None = None,
                kv_lens: torch.Tensor | None = None) -> torch.Tensor:
        assert q.shape[2] == self.n_heads and q.shape[3] == self.head_dim
        return window_attn(q, k, v, self.attn_sink, window=self.window, n_first=self.n_first,
                           kv_lens=kv_lens, softmax_scale=self.softmax_scale)

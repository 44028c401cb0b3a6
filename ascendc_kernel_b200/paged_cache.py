"""A paged key-value cache and the operators that write it, read it and shrink it.

The pool is ``k_pages`` and ``v_pages`` [num_pages, page_size, hk, d] (``v_pages`` None:
the keys serve as values, as in :mod:`ascendc_kernel_b200.sparse_attn`) and, where
eviction is wanted, ``weights`` [num_pages, page_size] fp32: the attention that each row
has gathered. ``block_table`` [b, max_pages] int32 names each sequence's pages.

* :func:`cache_append` -- new rows into the pages
* :func:`paged_attn`   -- one new token per sequence over the cache
* :func:`cache_evict`  -- the rows that gathered most attention move to fresh pages
* :class:`PagedKVCache` -- a pool with its tables and free pages, on which the three run

Shape preconditions are checked with ``assert``; CUDA-level failures raise DsaError.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from ._native import lib
from .window_attn import DTYPES, _ptr, _run, _sink_on, _strided, _strides


def _check_pool(k_pages, v_pages, weights, block_table):
    """Checks what the operators share; returns num_pages, page_size, hk, d and the device."""
    assert k_pages.is_cuda and k_pages.dtype in DTYPES and k_pages.dim() == 4, \
        "k_pages must be a CUDA tensor [num_pages, page_size, hk, d], bf16 or fp16"
    shape, dev = k_pages.shape, k_pages.device
    n, page, hk, d = shape
    for x in (k_pages, v_pages):
        if x is not None:
            assert x.shape == shape and x.dtype == k_pages.dtype and x.device == dev, \
                "v_pages must be like k_pages"
            assert x.data_ptr() % 16 == 0 and (x.is_contiguous() or (
                x.stride(3) == 1 and all(s % 8 == 0 and s > 0 for s in x.stride()[:3]))), \
                "pages need a contiguous head_dim and strides in multiples of 8 elements"
    assert n >= 1 and page >= 1 and page % 8 == 0, "page_size must be a multiple of 8"
    assert d in (64, 128), "kernel specialised to head_dim in (64, 128)"
    if weights is not None:
        assert weights.shape == shape[:2] and weights.dtype == torch.float32 \
            and weights.device == dev and weights.is_contiguous(), \
            "weights must be fp32 [num_pages, page_size], contiguous"
    _check_table(block_table, dev, "block_table")
    return n, page, hk, d, dev


def _check_table(table, dev, name):
    assert table.dtype == torch.int32 and table.dim() == 2 and table.device == dev \
        and table.shape[1] >= 1, f"{name} must be int32 [b, pages] on the pool's device"


def _check_lens(lens, b, dev, name="lens"):
    assert lens.dtype == torch.int32 and lens.shape == (b,) and lens.device == dev, \
        f"{name} must be int32 [b] on the pool's device"


class _NoGradient(torch.autograd.Function):
    """x, whose gradient is asked for in vain: better an error than a loss without its share."""

    @staticmethod
    def forward(ctx, x, *sources):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, dx):
        raise RuntimeError("paged_attn has no gradient: train with window_attn, or call it "
                           "under torch.no_grad()")


@functools.lru_cache(maxsize=256)
def _attn_workspace(b, h, hk, d, max_pages, page, weights) -> int:
    return max(lib().dsa_paged_attn_workspace_bytes(b, h, hk, d, max_pages, page, weights), 256)


def paged_attn(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor | None,
               block_table: torch.Tensor, lens: torch.Tensor, sink: torch.Tensor | None = None, *,
               window: int = 0, n_first: int = 0, softmax_scale: float | None = None,
               weights: torch.Tensor | None = None, out: torch.Tensor | None = None,
               return_lse: bool = False):
    """Attention of one new token per sequence over the cache, whose rows include it.

    q [b, h, d]; lens [b] int32 counts each sequence's rows. The token sees rows
    j < lens[b], with ``window`` > 0 only the last ``window`` and the first ``n_first`` of
    them; sink [h] fp32 logits or None; softmax_scale defaults to d ** -0.5. Returns out
    like q (0 where nothing is visible and there is no sink) and with ``return_lse`` the
    fp32 log of the softmax divisor [b, h]. With ``weights`` the slot of each visible row
    gains its attention weight summed over the heads, in place. The softmax's weights are
    rounded to q's type before they meet v, everything else is fp32. Not differentiable: a
    backward pass that reaches the results of a call with gradients raises RuntimeError.
    """
    assert q.dim() == 3, "q must be [b, h, d]"
    given = (q, k_pages, v_pages, sink)
    n, page, hk, d, dev = _check_pool(k_pages, v_pages, weights, block_table)
    b, h, _ = q.shape
    assert q.dtype == k_pages.dtype and q.device == dev and q.shape[2] == d, \
        "q must have the pool's type, device and head_dim"
    assert h % hk == 0 and 1 <= h // hk <= 128, \
        "n_heads must be a multiple of n_kv_heads, at most 128 to a group"
    width = block_table.shape[1]
    assert block_table.shape[0] == b
    _check_lens(lens, b, dev)
    scale = float(d ** -0.5 if softmax_scale is None else softmax_scale)
    assert window >= 0 and n_first >= 0 and scale > 0
    if sink is not None:
        assert sink.numel() == h, "sink must have n_heads entries"
        sink = _sink_on(sink, dev)
    strides = None
    if not q.is_contiguous():
        if q.stride(2) != 1 or any(m > 1 and (s <= 0 or s % 8)
                                   for m, s in zip(q.shape, q.stride()[:2])):
            q = q.contiguous()
        else:
            strides = (ctypes.c_int64 * 2)(*q.stride()[:2])
    if q.data_ptr() % 16:
        q, strides = q.clone(memory_format=torch.contiguous_format), None
    if out is None:
        out = torch.empty((b, h, d), dtype=q.dtype, device=dev)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == dev \
            and out.is_contiguous(), "out must be contiguous and like q"
    lse = torch.empty((b, h), dtype=torch.float32, device=dev) if return_lse else None
    table, lens = block_table.contiguous(), lens.contiguous()
    nbytes = _attn_workspace(b, h, hk, d, width, page, 0 if weights is None else 1)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    k_strides = _strides(k_pages)
    if v_pages is None:
        values, v_strides = k_pages.data_ptr(), k_strides
    else:
        values, v_strides = v_pages.data_ptr(), _strides(v_pages)
    _run("dsa_paged_attn_fwd", q.get_device(), q.data_ptr(), strides, k_pages.data_ptr(), k_strides,
         values, v_strides, table.data_ptr(), lens.data_ptr(), _ptr(sink), out.data_ptr(), _ptr(lse),
         _ptr(weights), DTYPES[q.dtype], b, h, hk, d, n, page, width, min(int(window), 1 << 28),
         min(int(n_first), 1 << 28), scale, ws.data_ptr(), nbytes)
    if torch.is_grad_enabled():
        sources = [x for x in given if x is not None and x.requires_grad]
        if sources:
            out = _NoGradient.apply(out, *sources)
            lse = _NoGradient.apply(lse, *sources) if return_lse else None
    return (out, lse) if return_lse else out


def cache_append(k: torch.Tensor, v: torch.Tensor | None, k_pages: torch.Tensor,
                 v_pages: torch.Tensor | None, block_table: torch.Tensor, start: torch.Tensor,
                 weights: torch.Tensor | None = None) -> None:
    """Writes k, v [b, t, hk, d] to rows start[b] .. start[b] + t - 1 of each sequence and
    sets their slots' ``weights`` to 0. ``start`` int32 [b]. Rows past the table's room or
    of pages that do not exist are not written (see ``_native.device_error``)."""
    n, page, hk, d, dev = _check_pool(k_pages, v_pages, weights, block_table)
    assert (v is None) == (v_pages is None), "v and v_pages are both given or both None"
    assert k.dim() == 4 and k.shape[2:] == k_pages.shape[2:] and k.dtype == k_pages.dtype \
        and k.device == dev, "k must be [b, t, hk, d] of the pool's type and device"
    b, t = k.shape[:2]
    assert block_table.shape[0] == b
    _check_lens(start, b, dev, "start")
    k = _strided(k)
    v_ptr = v_strides = None
    if v is not None:
        assert v.shape == k.shape and v.dtype == k.dtype and v.device == dev, "v must be like k"
        v = _strided(v)
        v_ptr, v_strides = v.data_ptr(), _strides(v)
    table, start = block_table.contiguous(), start.contiguous()
    _run("dsa_cache_append", k.get_device(), k.data_ptr(), _strides(k), v_ptr, v_strides,
         k_pages.data_ptr(), _strides(k_pages), _ptr(v_pages),
         None if v_pages is None else _strides(v_pages), _ptr(weights), table.data_ptr(),
         start.data_ptr(), b, t, hk, d, n, page, table.shape[1])


def cache_evict(k_pages: torch.Tensor, v_pages: torch.Tensor | None, weights: torch.Tensor,
                block_table: torch.Tensor, lens: torch.Tensor, dst_table: torch.Tensor, *,
                budget: int, n_first: int = 0, n_recent: int = 0):
    """Keeps at most ``budget`` rows of each sequence: the first ``n_first``, the last
    ``n_recent`` and, of those between, the ones with the largest weights (equal weights:
    the lower row). The kept rows and their weights are copied in ascending order to rows
    0, 1, ... of the pages of ``dst_table`` [b, dst_pages] int32 (distinct pages that no
    sequence of the call uses); the old pages stay as they are. Returns the kept rows
    [b, budget] int32, filled up with -1, and the new lengths [b] int32."""
    n, page, hk, d, dev = _check_pool(k_pages, v_pages, weights, block_table)
    b, width = block_table.shape
    assert weights is not None, "eviction goes by the weights"
    _check_lens(lens, b, dev)
    _check_table(dst_table, dev, "dst_table")
    assert dst_table.shape[0] == b
    assert budget >= 1 and n_first >= 0 and n_recent >= 0 and n_first + n_recent <= budget, \
        "n_first + n_recent <= budget"
    assert budget <= dst_table.shape[1] * page, "dst_table has no room for budget rows"
    table, lens, dst = block_table.contiguous(), lens.contiguous(), dst_table.contiguous()
    kept = torch.empty((b, budget), dtype=torch.int32, device=dev)
    left = torch.empty((b,), dtype=torch.int32, device=dev)
    _run("dsa_cache_evict", k_pages.get_device(), k_pages.data_ptr(), _strides(k_pages),
         _ptr(v_pages), None if v_pages is None else _strides(v_pages), weights.data_ptr(),
         table.data_ptr(), lens.data_ptr(), dst.data_ptr(), kept.data_ptr(), left.data_ptr(), b, hk,
         d, n, page, width, dst.shape[1], budget, n_first, n_recent)
    return kept, left


class PagedKVCache:
    """A pool of pages with the tables, lengths and free pages of a batch of sequences.

    Page numbers and lengths are kept on the host as well and go up from pinned memory, so no
    call waits for the GPU (the first ones may, while that memory is allocated); the pool is
    used on the caller's current stream, in call order. All sequences advance together: an
    ``append`` adds as many rows to each. ``shared`` holds one
    tensor that serves as keys and values; ``track_weights`` holds the attention each row
    gathers (needed for :meth:`evict`).
    """

    def __init__(self, batch: int, num_pages: int, page_size: int, max_len: int, n_kv_heads: int,
                 head_dim: int, *, shared: bool = False, track_weights: bool = False,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        assert page_size >= 8 and page_size % 8 == 0, "page_size must be a multiple of 8"
        assert batch >= 1 and num_pages >= 1 and max_len >= 1
        self.batch, self.page_size, self.max_len = batch, page_size, max_len
        shape = (num_pages, page_size, n_kv_heads, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = None if shared else torch.zeros(shape, dtype=dtype, device=device)
        self.weights = (torch.zeros(num_pages, page_size, dtype=torch.float32, device=device)
                        if track_weights else None)
        self.max_pages = -(-max_len // page_size)
        self.block_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.host_lens = [0] * batch
        self.pages = [[] for _ in range(batch)]
        self.free = list(range(num_pages - 1, -1, -1))

    def _take(self, count: int) -> list[int]:
        if count > len(self.free):
            raise RuntimeError(f"the page pool is exhausted: {count} pages wanted, "
                               f"{len(self.free)} free")
        taken = self.free[len(self.free) - count:][::-1]
        del self.free[len(self.free) - count:]
        return taken

    def _table(self, rows: list[list[int]], width: int) -> torch.Tensor:
        """The rows' page numbers on the host, in pinned memory where the pool is on a GPU: a
        copy from there need not be waited for (torch keeps the memory until it is done)."""
        return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32,
                            pin_memory=self.block_table.is_cuda)

    def append(self, k: torch.Tensor, v: torch.Tensor | None = None) -> None:
        """Adds the next rows k, v [batch, t, hk, d] of every sequence."""
        t = k.shape[1]
        assert k.shape[0] == self.batch
        need = []
        for i in range(self.batch):
            assert self.host_lens[i] + t <= self.max_len, "sequence longer than max_len"
            need.append(-(-(self.host_lens[i] + t) // self.page_size) - len(self.pages[i]))
        taken = self._take(sum(max(n, 0) for n in need))
        if taken:
            for i, n in enumerate(need):
                if n > 0:
                    self.pages[i] += taken[:n]
                    del taken[:n]
            self.block_table.copy_(self._table(self.pages, self.max_pages), non_blocking=True)
        cache_append(k, v, self.k_pages, self.v_pages, self.block_table, self.lens, self.weights)
        self.lens += t
        self.host_lens = [n + t for n in self.host_lens]

    def attend(self, q: torch.Tensor, sink: torch.Tensor | None = None, *, window: int = 0,
               n_first: int = 0, softmax_scale: float | None = None) -> torch.Tensor:
        """:func:`paged_attn` of q [batch, h, d] over the cache; the weights, where they are
        tracked, gain this step's attention."""
        return paged_attn(q, self.k_pages, self.v_pages, self.block_table, self.lens, sink,
                          window=window, n_first=n_first, softmax_scale=softmax_scale,
                          weights=self.weights)

    def evict(self, budget: int, n_first: int = 0, n_recent: int = 0) -> torch.Tensor:
        """:func:`cache_evict` of every sequence to at most ``budget`` rows. The old pages
        are free again; returns the kept rows [batch, budget] int32, filled up with -1."""
        assert self.weights is not None, "eviction needs track_weights"
        width = -(-budget // self.page_size)
        after = [min(n, budget) for n in self.host_lens]
        need = [-(-n // self.page_size) for n in after]
        taken, fresh, at = self._take(sum(need)), [], 0
        for n in need:
            fresh.append(taken[at:at + n])
            at += n
        try:
            dst = self._table(fresh, width).to(self.block_table.device, non_blocking=True)
            kept, left = cache_evict(self.k_pages, self.v_pages, self.weights, self.block_table,
                                     self.lens, dst, budget=budget, n_first=n_first,
                                     n_recent=n_recent)
        except Exception:
            self.free += taken[::-1]  # as _take found them
            raise
        self.host_lens = after
        for old in self.pages:
            self.free += old
        self.pages = fresh
        self.block_table.copy_(self._table(self.pages, self.max_pages), non_blocking=True)
        self.lens.copy_(left)
        return kept

"""Windowed attention and the paged cache at the ends of their ranges: chunks whose pages are
absent under very low scores, a pool whose calls must not wait for the GPU, losses that
use what has no gradient, chunks after prefixes of different lengths.

Bounds as in test_paged_cache_gpu.py; where scores are about -100, their fp32 sums (64 terms,
each addition off by at most 2^-23 of 800, times the scale of 1/8) are good to 8e-4, so the
fp32 part is 1e-3 of the magnitudes.
"""

import math

import pytest
import torch

from ascendc_kernel_b200 import _native
from ascendc_kernel_b200.paged_cache import PagedKVCache, paged_attn
from ascendc_kernel_b200.window_attn import window_attn

pytestmark = pytest.mark.gpu

DEVERR_CACHE = 0x0040


# rows, page, first and last + 1 page that is absent: the first chunk of 128 rows, one between
# others, the last one, all but one; chunks of their own block and blocks of several chunks
@pytest.mark.parametrize("rows,page,gone", [
    (300, 16, (0, 8)), (300, 16, (8, 16)), (300, 16, (16, 19)), (300, 16, (0, 16)),
    (60000, 64, (2, 4)), (60000, 64, (101, 460)),
])
@pytest.mark.parametrize("weighted", [False, True])
def test_absent_chunks_under_low_scores(cuda_device, rows, page, gone, weighted):
    """Rows without a page count as hidden, also where they fill whole chunks and every score
    lies far below 0."""
    h, d, dtype = 4, 64, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(7)
    width = -(-rows // page)
    k = torch.randn(width, page, 1, d, generator=g, device="cuda").to(dtype) * 0.25
    v = torch.randn(width, page, 1, d, generator=g, device="cuda").to(dtype)
    k[..., 0] = -100.0
    q = torch.randn(1, h, d, generator=g, device="cuda").to(dtype)
    q[..., 0] = 8.0
    table = torch.arange(width, dtype=torch.int32, device="cuda")[None].contiguous()
    table[0, gone[0]:gone[1]] = -1
    n = torch.full((1,), rows, dtype=torch.int32, device="cuda")
    weights = torch.zeros(width, page, device="cuda") if weighted else None
    out, lse = paged_attn(q, k, v, table, n, weights=weights, return_lse=True)
    assert _native.device_error(0) == DEVERR_CACHE
    live = torch.ones(width, page, dtype=torch.bool, device="cuda")
    live[gone[0]:gone[1]] = False
    live.view(-1)[rows:] = False
    kk, vv = k[live][:, 0].double(), v[live][:, 0].double()
    s = (q[0].double() @ kk.T) * d ** -0.5
    p = torch.softmax(s, 1)
    mag = p @ vv.abs()
    want = p @ vv
    assert s.max() < -90 and len(kk) > 0
    assert ((out[0].double() - want).abs() <= 2.0 ** -8 * (want.abs() + mag) + 1e-3 * mag).all()
    assert ((lse[0].double() - torch.logsumexp(s, 1)).abs() <= 1e-3).all()
    if weighted:
        assert not weights[~live].any()
        assert ((weights[live].double() - p.sum(0)).abs() <= 1e-3 * p.sum(0)).all()


def test_pool_calls_do_not_wait(cuda_device):
    """Appends that take pages and evictions while the stream is busy: torch reports a call that
    would wait, and the tables that they send arrive whole."""
    b, page, d = 2, 16, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(b, 60, 1, d, generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn(b, 4, d, generator=g, device="cuda").to(torch.bfloat16)

    def steps(c):
        for t in (60, 40, 1, 30):
            c.append(x[:, :t].contiguous())
            c.attend(q)
            c.evict(50, 2, 4)
            c.append(x[:, t - 1:t].contiguous())
        return c.attend(q), c.lens.clone()

    def pool():
        return PagedKVCache(b, 40, page, 200, 1, d, shared=True, track_weights=True)

    want, lens = steps(pool())
    busy = pool()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        torch.cuda._sleep(20_000_000)  # about 10 ms: every upload below is pending at once
        got, left = steps(busy)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(got, want) and torch.equal(left, lens)
    assert busy.lens.tolist() == busy.host_lens
    for i, pages in enumerate(busy.pages):
        assert busy.block_table[i].tolist() == pages + [-1] * (busy.max_pages - len(pages))


def test_a_loss_with_lse_is_refused(cuda_device):
    """lse has no gradient: a loss that uses it must not get one without its share."""
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k = (torch.randn(1, 20, h, 64, generator=g, device="cuda").to(torch.bfloat16)
            .requires_grad_(True) for h in (4, 2))
    sink = torch.randn(4, generator=g, device="cuda").requires_grad_(True)
    out, lse = window_attn(q, k, None, sink, window=9, return_lse=True)
    for loss in (out.float().sum() + lse.square().sum(), lse.sum()):
        with pytest.raises(RuntimeError, match="lse"):
            torch.autograd.grad(loss, (q, k, sink), retain_graph=True)
    # without it, and with it detached, nothing changes
    want = torch.autograd.grad(window_attn(q, k, None, sink, window=9).float().sum(), (q, k, sink))
    for loss in (out.float().sum(), out.float().sum() + lse.detach().sum()):
        for a, b in zip(torch.autograd.grad(loss, (q, k, sink), retain_graph=True), want):
            assert torch.equal(a, b)


def test_a_loss_over_the_cache_is_refused(cuda_device):
    """Single-token attention has no gradient: neither q's nor the sink's graph ends silently."""
    g = torch.Generator(device="cuda").manual_seed(8)
    k = torch.randn(3, 16, 1, 64, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None].contiguous()
    n = torch.full((1,), 40, dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    sink = torch.randn(4, generator=g, device="cuda")
    want, want_lse = paged_attn(q, k, None, table, n, sink, return_lse=True)
    assert not want.requires_grad and not want_lse.requires_grad
    for leaf in ("q", "sink", "noncontiguous q", "fp64 sink"):
        a, s = q.clone(), sink.clone()
        x = s if "sink" in leaf else a
        x.requires_grad_(True)
        if leaf == "fp64 sink":
            s = s.double()
        if leaf == "noncontiguous q":
            a = a.transpose(1, 2).contiguous().transpose(1, 2)
        buffer = torch.empty_like(q)
        for kw in (dict(), dict(out=buffer)):
            out, lse = paged_attn(a, k, None, table, n, s, return_lse=True, **kw)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
            for y in (out, lse):
                with pytest.raises(RuntimeError, match="no gradient"):
                    (x.float().sum() + y.float().sum()).backward()
            with torch.no_grad():
                assert not paged_attn(a, k, None, table, n, s, **kw).requires_grad
        assert torch.equal(buffer, want)


def test_a_chunk_after_prefixes_of_different_lengths(cuda_device):
    """kv_lens hides keys and moves no query: of a padded batch, a chunk's queries stand where
    the padded length puts them. A call per length, on keys cut to it, is the chunk of that
    sequence's own whole prompt."""
    m, h, hk, d, n, lens = 40, 6, 2, 64, 300, [300, 137, 45, 40]
    g = torch.Generator(device="cuda").manual_seed(9)
    whole = torch.randn(4, n, h, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(4, n, hk, d, generator=g, device="cuda").to(torch.bfloat16)
            for _ in range(2))
    kw = dict(window=60, n_first=3)
    full = window_attn(whole, k, v, kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                       **kw)  # whole prompts, padded on the right
    for i, x in enumerate(lens):
        rows = slice(x - m, x)
        got = window_attn(whole[i:i + 1, rows], k[i:i + 1, :x], v[i:i + 1, :x], **kw)
        # the rounding of the softmax's weights depends on how the keys are cut into blocks:
        # both sides are within u (|out| + sum P |v|) of the definition
        scale = v[i, :x].abs().max().double()
        assert ((got[0].double() - full[i, rows].double()).abs() <= 2 * 2.0 ** -8 * 2 * scale).all()
    # the padded form is another thing: the second sequence's queries stand past its keys
    n_i = torch.tensor([lens[1]], dtype=torch.int32, device="cuda")
    far = window_attn(whole[1:2, :m], k[1:2], v[1:2], kv_lens=n_i, **kw)
    want = window_attn(whole[1:2, :1], k[1:2, :3], v[1:2, :3], window=3)
    assert ((far[0, 0].double() - want[0, 0].double()).abs() <= 2.0 ** -6 * v.abs().max()).all()

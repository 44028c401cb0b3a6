"""The paged cache: append, single-token attention and eviction, against plain forms.

Attention bounds as in test_window_attn_gpu.py: u (|out| + sum P |v|) for the two roundings,
1e-4 of the magnitudes for fp32, and one subnormal step of fp16 weights a key. Append and
evict copy: they are exact.
"""

import math

import pytest
import torch

from ascendc_kernel_b200 import _native
from ascendc_kernel_b200.paged_cache import PagedKVCache, cache_append, cache_evict, paged_attn

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -17}
F32 = 1e-4
DEVERR_CACHE = 0x0040


def pool(b, max_len, page, hk, d, dtype, shared, seed=0, spare=3):
    """A pool in shuffled page order whose unused slots hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = -(-max_len // page)
    n = b * width + spare
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    k = torch.full((n, page, hk, d), math.nan, dtype=dtype, device="cuda")
    v = None if shared else torch.full_like(k, math.nan)
    return k, v, order[:b * width].reshape(b, width), order[b * width:], g


def fill(k, v, table, lens, g):
    page = k.shape[1]
    rows = []
    for i, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        at = table[i].long()[j // page], j % page
        pair = []
        for x in (k, v):
            if x is not None:
                r = torch.randn(n, *k.shape[2:], generator=g, device="cuda").to(k.dtype)
                x[at] = r
                pair.append(r)
        rows.append((pair[0], pair[-1], at))
    return rows


def definition(q, keys, values, sink, window, n_first, scale):
    """One sequence: q [h, d], keys and values [n, hk, d]; out, lse, P, magnitudes."""
    h, d = q.shape
    n, hk = keys.shape[:2]
    j = torch.arange(n, device=q.device)
    see = torch.ones(n, dtype=torch.bool, device=q.device)
    if window:
        see = (j >= n - window) | (j < n_first)
    kk = keys.double().repeat_interleave(h // hk, 1).transpose(0, 1)
    vv = values.double().repeat_interleave(h // hk, 1).transpose(0, 1)
    s = (kk @ q.double()[:, :, None])[..., 0] * scale
    s = s.masked_fill(~see, -math.inf)
    s2 = s if sink is None else torch.cat([s, sink.double()[:, None]], 1)
    lse = torch.logsumexp(s2, 1) if s2.shape[1] else torch.full((h,), -math.inf, device=q.device)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    out = (p[:, None] @ vv)[:, 0]
    return out, lse, p, (p[:, None] @ vv.abs())[:, 0], (see.double() @ vv.abs())


# lens, page, h, hk, window, n_first: one row; page ends inside a chunk and a chunk inside
# a page; groups of 1, 3, 64, an odd one above 64 and 128; empty sequences among others;
# windows across page borders, first tokens beside and inside them; more sequences than
# a warp has lanes; a long one beside short ones
CASES = [
    ([1], 8, 1, 1, 0, 0), ([333], 64, 64, 1, 0, 0), ([0, 700, 5, 0], 24, 24, 8, 0, 0),
    ([129, 1000, 63], 16, 12, 2, 100, 4), ([1500, 257], 128, 128, 1, 0, 0),
    ([900, 31], 64, 77, 1, 300, 130), ([513, 40], 40, 4, 4, 1, 1), ([200, 199], 32, 2, 1, 33, 200),
    ([3 + 7 * i for i in range(40)], 32, 33, 1, 17, 3), ([9000, 1, 0, 130], 40, 8, 2, 0, 0),
    # several pieces and tens of chunks to each block of the split kernel
    ([5000, 625, 4200, 3111, 2000, 901, 4999], 64, 32, 8, 0, 0), ([30000, 29000], 16, 64, 1, 0, 0),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16),
                                     (64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("sink,shared", [(True, True), (False, False)])
def test_paged_attention(cuda_device, case, d, dtype, sink, shared):
    lens, page, h, hk, window, first = case
    b = len(lens)
    k, v, table, _, g = pool(b, max(lens) + 9, page, hk, d, dtype, shared)
    rows = fill(k, v, table, lens, g)
    q = torch.randn(b, h, d, generator=g, device="cuda").to(dtype)
    s = torch.randn(h, generator=g, device="cuda") * 3 if sink else None
    weights = torch.rand(k.shape[:2], generator=g, device="cuda") * 5
    want_w, tol_w = weights.double(), 2.0 ** -22 * weights.double()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    before = weights.clone()
    out, lse = paged_attn(q, k, v, table, n, s, window=window, n_first=first, weights=weights,
                          return_lse=True)
    plain = paged_attn(q, k, v, table, n, s, window=window, n_first=first)
    assert torch.equal(out, plain), "with and without weights, and from call to call"
    assert torch.isfinite(out).all()
    for i in range(b):
        o, l, p, mag, keys = definition(q[i], rows[i][0], rows[i][1], s, window, first, d ** -0.5)
        bound = U[dtype] * (o.abs() + mag) + F32 * mag + TINY[dtype] * (keys + 1)
        assert ((out[i].double() - o).abs() <= bound).all()
        dead = l == -math.inf
        assert torch.equal(lse[i] == -math.inf, dead)
        assert ((lse[i].double() - l)[~dead].abs() <= F32 * (1 + l[~dead].abs())).all()
        want_w[rows[i][2]] += p.sum(0)
        tol_w[rows[i][2]] += F32 * p.sum(0)
    assert ((weights.double() - want_w).abs() <= tol_w).all()
    untouched = want_w == before.double()
    assert torch.equal(weights[untouched], before[untouched])
    assert _native.device_error(0) == 0


def test_attention_with_climbing_scores_and_strided_pages(cuda_device):
    """Scores that climb by hundreds along the cache move the references; the pool is a view
    of one buffer with K and V side by side; the call runs on another stream."""
    lens, page, h, hk, d = [2000, 700], 16, 8, 2, 64
    both = torch.zeros(300, page, 2, hk, d, device="cuda", dtype=torch.bfloat16)
    k, v = both[:, :, 0], both[:, :, 1]
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randperm(300, generator=g, device="cuda")[:250].to(torch.int32).reshape(2, 125)
    rows = fill(k, v, table, lens, g)
    q = torch.randn(2, h, d, generator=g, device="cuda").to(torch.bfloat16)
    q[..., 0] = 8.0
    for i, n in enumerate(lens):
        climb = torch.linspace(-100, 100, n, device="cuda").to(torch.bfloat16)
        k[rows[i][2][0], rows[i][2][1], :, 0] = climb[:, None]
        rows[i][0][:, :, 0] = climb[:, None]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = torch.stack([q, q], 2)[:, :, 0]  # every other row of a buffer
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = paged_attn(qs, k, v, table, n)
    torch.cuda.synchronize()
    for i in range(2):
        o, _, _, mag, _ = definition(q[i], rows[i][0], rows[i][1], None, 0, 0, d ** -0.5)
        bound = (2.0 ** -8 + 2.0 ** -12) * (o.abs() + mag)
        assert ((out[i].double() - o).abs() <= bound).all()


def test_pages_past_32_bits(cuda_device):
    """A page whose offset is above 2^32 bytes."""
    page, hk, d = 64, 1, 128
    count = 2 ** 33 // (page * hk * d * 2) + 2
    k = torch.empty(count, page, hk, d, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(count, page, device="cuda")
    table = torch.tensor([[count - 1, 0]], dtype=torch.int32, device="cuda")
    x = torch.randn(1, 100, hk, d, device="cuda").to(torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache_append(x, None, k, None, table, zero, w)
    assert torch.equal(k[count - 1], x[0, :64]) and torch.equal(k[0, :36], x[0, 64:])
    q = torch.randn(1, 4, d, device="cuda").to(torch.bfloat16)
    n = torch.full((1,), 100, dtype=torch.int32, device="cuda")
    small, wsmall = torch.stack([k[count - 1], k[0], k[0]]), torch.zeros(3, page, device="cuda")
    t2 = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    assert torch.equal(paged_attn(q, k, None, table, n, weights=w),
                       paged_attn(q, small, None, t2, n, weights=wsmall))
    assert torch.equal(w[count - 1], wsmall[0]) and torch.equal(w[0], wsmall[1])
    dst = torch.tensor([[count - 2]], dtype=torch.int32, device="cuda")
    kept, left = cache_evict(k, None, w, table, n, dst, budget=20)
    assert left.item() == 20 and torch.equal(k[count - 2, :20], x[0, kept[0].long()])


def test_table_entries_that_name_no_page(cuda_device):
    """Their rows count as hidden and the error word says so; nothing is read or written
    there. Lengths past the table's room are clamped."""
    page, d = 16, 64
    k, v, table, _, g = pool(1, 64, page, 1, d, torch.bfloat16, False)
    rows = fill(k, v, table, [64], g)
    bad = table.clone()
    bad[0, 1], bad[0, 2] = -1, k.shape[0]
    q = torch.randn(1, 2, d, generator=g, device="cuda").to(torch.bfloat16)
    n = torch.full((1,), 64, dtype=torch.int32, device="cuda")
    out = paged_attn(q, k, v, bad, n)
    assert _native.device_error(0) == DEVERR_CACHE
    live = list(range(16)) + list(range(48, 64))
    o, _, _, mag, _ = definition(q[0], rows[0][0][live], rows[0][1][live], None, 0, 0, d ** -0.5)
    assert ((out[0].double() - o).abs() <= (U[torch.bfloat16] + F32) * (o.abs() + mag)).all()
    assert torch.equal(paged_attn(q, k, v, table, n + 100), paged_attn(q, k, v, table, n))
    assert _native.device_error(0) == DEVERR_CACHE
    x = torch.ones(1, 8, 1, d, device="cuda", dtype=torch.bfloat16)
    was_k, was_v = k.clone(), v.clone()
    cache_append(x, x, k, v, bad, n - 44, None)   # rows 20 .. 27: page -1
    cache_append(x, x, k, v, bad, n, None)        # rows past the room
    cache_append(x, x, k, v, bad, n - 74, None)   # rows -10 .. -3
    assert _native.device_error(0) == DEVERR_CACHE
    for a, c in ((was_k, k), (was_v, v)):
        assert torch.equal(a.view(torch.int16), c.view(torch.int16))


def evict_plain(weights, table, lens, page, budget, first, recent):
    out = []
    for i, n in enumerate(lens):
        rows = list(range(n))
        if n > budget:
            w = [weights[table[i][j // page], j % page].item() for j in rows]
            middle = rows[first:n - recent]
            # NaN above all, equal weights by row
            middle.sort(key=lambda j: (0 if math.isnan(w[j]) else 1, -w[j] if w[j] == w[j] else 0, j))
            rows = rows[:first] + middle[:budget - first - recent] + rows[n - recent:]
        out.append(sorted(rows))
    return out


@pytest.mark.parametrize("lens,page,hk,d,budget,first,recent", [
    ([40, 33, 34, 0, 1], 8, 1, 64, 33, 0, 33), ([64, 65, 300], 16, 2, 64, 64, 3, 3),
    ([1000, 999], 24, 1, 128, 100, 4, 16), ([2600], 64, 1, 128, 1024, 4, 128),
    ([50, 70], 16, 3, 128, 1, 0, 0), ([50, 70], 16, 1, 64, 1, 1, 0), ([5000], 16, 1, 64, 4999, 0, 0),
])
@pytest.mark.parametrize("kind", ["ties", "spread", "special"])
def test_evict(cuda_device, lens, page, hk, d, budget, first, recent, kind):
    b = len(lens)
    width = -(-budget // page)
    k, v, table, spare, g = pool(b, max(max(lens), 1), page, hk, d, torch.bfloat16, False,
                                 spare=b * (width + 1))
    fill(k, v, table, lens, g)
    dst = spare[:b * (width + 1)].reshape(b, width + 1)  # a page more than needed
    weights = torch.rand(k.shape[:2], generator=g, device="cuda")
    if kind == "ties":
        weights = (weights * 3).floor() - 1  # negative, zero and positive, many alike
    elif kind == "special":
        pick = (torch.rand(k.shape[:2], generator=g, device="cuda") * 8).long()
        table_of = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42, 1.0],
                                device="cuda")
        weights = table_of[pick]
    was = weights.clone()
    wants = evict_plain(weights.cpu(), table.cpu(), lens, page, budget, first, recent)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    was_k, was_v = k.clone(), v.clone()
    kept, left = cache_evict(k, v, weights, table, n, dst, budget=budget, n_first=first,
                             n_recent=recent)
    same = torch.ones(k.shape[0], dtype=torch.bool, device="cuda")
    same[dst.long()] = False
    for a, c in ((was_k, k), (was_v, v)):
        assert torch.equal(a[same].view(torch.int16), c[same].view(torch.int16)), "old pages stay"
    for i, want in enumerate(wants):
        assert left[i].item() == len(want)
        assert kept[i].tolist() == want + [-1] * (budget - len(want))
        src = torch.tensor(want, dtype=torch.long, device="cuda")
        at = torch.arange(len(want), device="cuda")
        sp, dp = table[i].long()[src // page], dst[i].long()[at // page]
        for a, c in ((was_k, k), (was_v, v)):
            assert torch.equal(a[sp, src % page].view(torch.int16),
                               c[dp, at % page].view(torch.int16))
        assert torch.equal(was[sp, src % page].view(torch.int32),
                           weights[dp, at % page].view(torch.int32))
        rest = torch.arange(len(want), (width + 1) * page, device="cuda")
        assert not weights[dst[i].long()[rest // page], rest % page].any(), "free slots weigh 0"
    assert _native.device_error(0) == 0


@pytest.mark.parametrize("shared", [True, False])
def test_cache_lives_through_append_attend_evict(cuda_device, shared):
    """The class against a dense mirror of what every sequence still holds."""
    b, page, hk, h, d, first, recent, budget = 3, 16, 2, 6, 64, 2, 8, 40
    cache = PagedKVCache(b, 40, page, 200, hk, d, shared=shared, track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(2)
    keys = [torch.zeros(0, hk, d, device="cuda", dtype=torch.bfloat16)] * b
    values = list(keys)
    gained = [torch.zeros(0, device="cuda", dtype=torch.float64)] * b
    for step, t in enumerate([50, 1, 1, 13, 1, 20, 1, 1]):
        x = torch.randn(b, t, 2 * hk, d, generator=g, device="cuda").to(torch.bfloat16)
        cache.append(x[:, :, :hk], None if shared else x[:, :, hk:])
        q = torch.randn(b, h, d, generator=g, device="cuda").to(torch.bfloat16)
        out = cache.attend(q)
        for i in range(b):
            keys[i] = torch.cat([keys[i], x[i, :, :hk]])
            values[i] = torch.cat([values[i], x[i, :, :hk] if shared else x[i, :, hk:]])
            o, _, p, mag, _ = definition(q[i], keys[i], values[i], None, 0, 0, d ** -0.5)
            assert ((out[i].double() - o).abs() <= (2.0 ** -8 + F32) * (o.abs() + mag)).all()
            gained[i] = torch.cat([gained[i], torch.zeros(t, device="cuda").double()]) + p.sum(0)
        if step in (3, 5):
            kept = cache.evict(budget, first, recent)
            for i in range(b):
                rows = kept[i].long()
                rows = rows[rows >= 0]
                assert len(rows) == budget == cache.host_lens[i]
                keys[i], values[i], gained[i] = keys[i][rows], values[i][rows], gained[i][rows]
    assert cache.lens.tolist() == cache.host_lens == [len(x) for x in keys]
    used = [p for x in cache.pages for p in x]
    assert sorted(used + cache.free) == list(range(40)), "every page is used once or free"
    assert _native.device_error(0) == 0


def test_example_runs(cuda_device):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "window_cache.py")
    spec = importlib.util.spec_from_file_location("window_cache_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main()
    assert r["loss_after"] < r["loss_before"]
    assert torch.isfinite(r["last"]).all()
    assert max(r["lengths"]) <= 512 and r["lengths"][-1] < 300 + 64
    assert _native.device_error(0) == 0


def test_refusals(cuda_device):
    k, v, table, spare, g = pool(2, 64, 16, 2, 64, torch.bfloat16, False)
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    n = torch.full((2,), 5, dtype=torch.int32, device="cuda")
    w = torch.zeros(k.shape[:2], device="cuda")
    ok = dict(q=q, k_pages=k, v_pages=v, block_table=table, lens=n)
    for kw in (dict(q=q.float()), dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[:1]),
               dict(k_pages=k[:, :15]), dict(v_pages=v[:1]), dict(block_table=table.long()),
               dict(lens=n.long()), dict(lens=n[:1]), dict(window=-1), dict(softmax_scale=-1.0),
               dict(weights=w[:1]), dict(weights=w.double()), dict(sink=torch.zeros(3)),
               dict(k_pages=k[..., ::2], v_pages=None)):
        with pytest.raises(AssertionError):
            paged_attn(**{**ok, **kw})
    x = torch.zeros(2, 3, 2, 64, device="cuda", dtype=torch.bfloat16)
    for a in ((x, None, k, v, table, n), (x.half(), x.half(), k, v, table, n),
              (x[:, :, :1], x[:, :, :1], k, v, table, n), (x, x, k, v, table, n.long())):
        with pytest.raises(AssertionError):
            cache_append(*a)
    dst = spare[:2].reshape(2, 1)
    for kw in (dict(budget=17), dict(budget=0), dict(budget=8, n_first=5, n_recent=4),
               dict(budget=8, n_first=-1)):
        with pytest.raises(AssertionError):
            cache_evict(k, v, w, table, n, dst, **kw)
    cache = PagedKVCache(1, 2, 16, 64, 1, 64)
    one = torch.zeros(1, 33, 1, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.append(one, one)
    with pytest.raises(AssertionError):
        cache.append(torch.zeros(1, 65, 1, 64, device="cuda", dtype=torch.bfloat16), None)
    with pytest.raises(AssertionError):
        cache.evict(8)

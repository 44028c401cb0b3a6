"""Cases of the windowed attention and of the paged key-value cache, with their plain forms.

Four operators: attention with a sliding window and a few first tokens that stay visible
(``window_attn``; prompts and training steps), attention of one new token over a paged cache
(``paged_attn``), eviction from that cache by accumulated attention weight (``cache_evict``) and
the writing of new rows into it (``cache_append``).

With ``own`` false, ``run`` computes the plain form: torch operations on fp32 values, rounded
once at the end. With ``own`` true it calls this package. ``exact`` is the definition in fp64.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the framework's own attention batch (8 x 2600 tokens, 64 heads over one kv head that
        # serves as keys and values) under its model's window of 128
        dict(name="window_batch", kind="window", b=8, m=2600, n=2600, h=64, hk=1, d=128,
             window=128, first=4, sink=True, shared=True, ragged=False, dtype="bf16"),
        # a long prompt in grouped heads, window 4096
        dict(name="window_prompt", kind="window", b=1, m=16384, n=16384, h=32, hk=8, d=128,
             window=4096, first=4, sink=False, shared=False, ragged=False, dtype="bf16"),
        # the next chunk of prompts of different lengths, three heads to a group, 64 wide, fp16
        dict(name="window_chunk_ragged", kind="window", b=3, m=515, n=4611, h=24, hk=8, d=64,
             window=1000, first=7, sink=False, shared=False, ragged=True, dtype="fp16"),
        # training steps (forward, then all gradients): grouped heads, and the shared kv head
        dict(name="train_grouped", kind="train", b=2, m=4096, n=4096, h=32, hk=8, d=128,
             window=1024, first=4, sink=False, shared=False, ragged=False, dtype="bf16"),
        dict(name="train_shared", kind="train", b=2, m=2600, n=2600, h=64, hk=1, d=128,
             window=128, first=4, sink=True, shared=True, ragged=False, dtype="bf16"),
        # one user's next token early in a conversation: latency counts
        dict(name="decode_short", kind="decode", b=1, length=333, h=64, hk=1, d=128, page=64,
             window=0, first=0, sink=True, shared=True, weights=False, dtype="bf16"),
        # a serving batch of conversations of different lengths that tracks what to evict
        dict(name="decode_batch", kind="decode", b=64, length=8192, h=32, hk=8, d=128, page=64,
             window=0, first=0, sink=False, shared=False, weights=True, dtype="bf16"),
        # a few very long contexts on the shared kv head
        dict(name="decode_long_shared", kind="decode", b=8, length=131072, h=64, hk=1, d=128,
             page=64, window=0, first=0, sink=True, shared=True, weights=False, dtype="bf16"),
        # eviction from one conversation of the framework's length, and from a serving batch
        dict(name="evict_one", kind="evict", b=1, length=2600, hk=1, d=128, page=64, budget=1024,
             first=4, recent=128, shared=True, dtype="bf16"),
        dict(name="evict_batch", kind="evict", b=32, length=16384, hk=8, d=128, page=64,
             budget=4096, first=4, recent=512, shared=False, dtype="bf16"),
        # the new token of every sequence of a batch, and the rows of a few prompts
        dict(name="append_step", kind="append", b=64, t=1, length=8192, hk=8, d=128, page=64,
             shared=False, dtype="bf16"),
        dict(name="append_prompt", kind="append", b=4, t=4096, length=8192, hk=8, d=128, page=64,
             shared=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    hk = rng.choice([1, 1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 6, 7, 8, 16, 32, 64, 128])
    return min(g, 128 // hk) * hk, hk


def draw(rng):
    kind = rng.choice(["window", "window", "train", "train", "decode", "decode", "decode", "evict",
                       "evict", "append"])
    limit = max((work(c)["flops"], work(c)["bytes"]) for c in listed() if c["kind"] == kind)
    most = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
    while True:
        h, hk = _heads(rng)
        d, dtype = rng.choice([64, 128]), rng.choice(["bf16", "bf16", "fp16"])
        if kind in ("window", "train"):
            n = _log(rng, 16, 16384 if kind == "window" else 4096)
            m = n if rng.random() < 0.7 else _log(rng, 1, n)
            case = dict(kind=kind, b=_log(rng, 1, 8), m=m, n=n, h=h, hk=hk, d=d,
                        window=_log(rng, 8, 4096), first=rng.choice([0, 1, 4, 7, 130]),
                        sink=rng.random() < 0.5, shared=rng.random() < 0.4,
                        ragged=rng.random() < 0.4, dtype=dtype)
        elif kind == "decode":
            whole = rng.random() < 0.6
            case = dict(kind=kind, b=_log(rng, 1, 64), length=_log(rng, 16, 131072), h=h, hk=hk,
                        d=d, page=rng.choice([16, 24, 64, 128]),
                        window=0 if whole else _log(rng, 8, 4096),
                        first=0 if whole else rng.choice([0, 4, 130]), sink=rng.random() < 0.5,
                        shared=rng.random() < 0.4, weights=rng.random() < 0.4, dtype=dtype)
        elif kind == "evict":
            length = _log(rng, 64, 32768)
            budget = _log(rng, 32, max(33, length // 2))
            first = rng.choice([0, 4, 16])
            case = dict(kind=kind, b=_log(rng, 1, 32), length=length, hk=hk, d=d,
                        page=rng.choice([16, 24, 64, 128]), budget=budget, first=first,
                        recent=min(budget - first, rng.choice([0, 16, 100, 512])),
                        shared=rng.random() < 0.4, dtype=dtype)
        else:
            t = _log(rng, 1, 4096)
            case = dict(kind=kind, b=_log(rng, 1, 64), t=t, length=_log(rng, t, 16384), hk=hk, d=d,
                        page=rng.choice([16, 24, 64, 128]), shared=rng.random() < 0.4, dtype=dtype)
        w = work(case)
        if w["flops"] <= limit[0] and w["bytes"] <= most and _pool_rows(case) * hk * d <= 2 ** 31:
            return case


def _lengths(case):
    """Lengths of the sequences: the first is whole, the others spread over an eighth to all."""
    full = case["n"] if "n" in case else case["length"]
    if "n" in case and not case["ragged"]:
        return [full] * case["b"]
    least = case.get("t", 1)
    return [max(least, int(full * (1.0 - 0.875 * ((i * 0.6180339887) % 1.0))))
            for i in range(case["b"])]


def _pages(case):
    return -(-case["length"] // case["page"]) if "length" in case else 0


def _pool_rows(case):
    if "length" not in case:
        return 0
    fresh = -(-case["budget"] // case["page"]) if case["kind"] == "evict" else 0
    return case["b"] * (_pages(case) + fresh) * case["page"]


def _pairs(case):
    """Visible (query, key) pairs of one head, summed over the batch."""
    total = 0
    for length in _lengths(case):
        for p in range(case["n"] - case["m"], case["n"]):
            lo = max(0, p - case["window"] + 1)
            total += max(0, min(p + 1, length) - lo) + min(case["first"], lo, length)
    return total


def _visible(case):
    """Visible keys of every sequence's new token."""
    out = []
    for length in _lengths(case):
        lo = max(0, length - case["window"]) if case["window"] else 0
        out.append(length - lo + min(case["first"], lo))
    return out


def work(case):
    kind, d, hk = case["kind"], case["d"], case["hk"]
    kv = 1 if case["shared"] else 2
    if kind in ("window", "train"):
        q = 2 * case["b"] * case["m"] * case["h"] * d
        k = 2 * kv * case["b"] * case["n"] * hk * d
        flops = _pairs(case) * case["h"] * d
        if kind == "window":
            return {"bytes": 2 * q + k, "flops": 4 * flops}
        # out is written and read again; dout is read, dq and the kv gradients are written
        return {"bytes": 2 * (2 * q + k) + q, "flops": 14 * flops}
    if kind == "decode":
        keys = sum(_visible(case))
        return {"bytes": 2 * kv * keys * hk * d + 4 * case["b"] * case["h"] * d
                + (8 * keys if case["weights"] else 0),
                "flops": 4 * keys * case["h"] * d}
    if kind == "evict":
        lengths = _lengths(case)
        kept = sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": 4 * sum(lengths) + kept * (2 * 2 * kv * hk * d + 8), "flops": sum(lengths)}
    rows = case["b"] * case["t"]
    return {"bytes": 2 * 2 * kv * rows * hk * d, "flops": rows}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    b, hk, d = case["b"], case["hk"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dt)

    st = {"case": case}
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    if case["kind"] in ("window", "train"):
        st["q"] = normal(b, case["m"], case["h"], d)
        st["k"] = normal(b, case["n"], hk, d)
        st["v"] = None if case["shared"] else normal(b, case["n"], hk, d)
        st["sink"] = (torch.randn(case["h"], generator=gen, device=dev) if case["sink"] else None)
        st["lens"] = lens if case["ragged"] else None
        if case["kind"] == "train":
            st["dout"] = normal(b, case["m"], case["h"], d)
            for x in ("q", "k", "v", "sink"):
                if st[x] is not None:
                    st[x].requires_grad_(True)
        return st
    # the cache: pages in shuffled order, every sequence with room for its longest length
    page, pages = case["page"], _pages(case)
    fresh = -(-case["budget"] // page) if case["kind"] == "evict" else 0
    count = b * (pages + fresh)
    order = torch.randperm(count, generator=gen, device=dev).to(torch.int32)
    st["table"] = order[:b * pages].reshape(b, pages).contiguous()
    st["lens"] = lens
    st["k_pages"] = normal(count, page, hk, d)
    st["v_pages"] = None if case["shared"] else normal(count, page, hk, d)
    if case["kind"] == "decode":
        st["q"] = normal(b, case["h"], d)
        st["sink"] = (torch.randn(case["h"], generator=gen, device=dev) if case["sink"] else None)
    if case["kind"] == "evict":
        st["dst"] = order[b * pages:].reshape(b, fresh).contiguous()
    if case["kind"] == "append":
        st["k"] = normal(b, case["t"], hk, d)
        st["v"] = None if case["shared"] else normal(b, case["t"], hk, d)
        st["start"] = lens - case["t"]
    if case["kind"] in ("evict", "append") or case["weights"]:
        # attention weights gathered over earlier steps: heavy-tailed, many alike near zero
        w = torch.rand(count, page, generator=gen, device=dev)
        st["weights"] = torch.round(w ** 8 * 4096) / 64
    else:
        st["weights"] = None
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    return {"window": _window, "train": _train, "decode": _decode, "evict": _evict,
            "append": _append}[kind](state)


def _window(st):
    c = st["case"]
    if own:
        from ascendc_kernel_b200.window_attn import window_attn
        return window_attn(st["q"], st["k"], st["v"], st["sink"], window=c["window"],
                           n_first=c["first"], kv_lens=st["lens"])
    return _plain_forward(st)[0]


def _train(st):
    c = st["case"]
    leaves = [st[x] for x in ("q", "k", "v", "sink") if st[x] is not None]
    if own:
        from ascendc_kernel_b200.window_attn import window_attn
        out = window_attn(st["q"], st["k"], st["v"], st["sink"], window=c["window"],
                          n_first=c["first"], kv_lens=st["lens"])
        return [out.detach(), *torch.autograd.grad(out, leaves, st["dout"])]
    with torch.no_grad():
        out, lse = _plain_forward(st)
        return [out, *_plain_backward(st, out, lse)]


def _blocks(c):
    """Blocks of queries with the keys that any of them sees (positions, on the host)."""
    step = 256
    for t0 in range(0, c["m"], step):
        t1 = min(t0 + step, c["m"])
        p0, p1 = t0 + c["n"] - c["m"], t1 - 1 + c["n"] - c["m"]
        lo = max(0, p0 - c["window"] + 1)
        yield t0, t1, p0, p1, min(c["first"], lo), lo


def _block_keys(x, first, lo, hi):
    """Rows [0, first) and [lo, hi) of x [b, n, hk, d], fp32 [b, hk, keys, d]."""
    return torch.cat([x[:, :first], x[:, lo:hi]], 1).float().transpose(1, 2)


def _block_rows(x, t0, t1, hk):
    """Rows of x [b, m, h, d], fp32 [b, hk, tokens * group, d]."""
    b, _, h, d = x.shape
    y = x[:, t0:t1].float().reshape(b, t1 - t0, hk, h // hk, d)
    return y.transpose(1, 2).reshape(b, hk, (t1 - t0) * (h // hk), d)


def _block_mask(st, c, p0, p1, first, lo):
    """Visible [b or 1, 1, tokens * group, keys]."""
    dev = st["q"].device
    pos = torch.arange(p0, p1 + 1, device=dev).repeat_interleave(c["h"] // c["hk"])[:, None]
    key = torch.cat([torch.arange(first, device=dev), torch.arange(lo, p1 + 1, device=dev)])
    vis = ((key <= pos) & ((key > pos - c["window"]) | (key < c["first"])))[None, None]
    if st["lens"] is not None:
        vis = vis & (key < st["lens"][:, None])[:, None, None, :]
    return vis


def _plain_forward(st):
    c, hk = st["case"], st["case"]["hk"]
    b, m, h, d = st["q"].shape
    g = h // hk
    out = torch.empty_like(st["q"], requires_grad=False)
    lse = torch.empty(b, hk, m, g, dtype=torch.float32, device=out.device)
    for t0, t1, p0, p1, first, lo in _blocks(c):
        rows = _block_rows(st["q"], t0, t1, hk) * d ** -0.5
        ks = _block_keys(st["k"], first, lo, p1 + 1)
        vs = ks if st["v"] is None else _block_keys(st["v"], first, lo, p1 + 1)
        s = rows @ ks.transpose(2, 3)
        s = s.masked_fill(~_block_mask(st, c, p0, p1, first, lo), -math.inf)
        top = s.amax(-1, keepdim=True)
        if st["sink"] is not None:
            sink = st["sink"].detach().reshape(hk, 1, g).expand(hk, t1 - t0, g).reshape(1, hk, -1, 1)
            top = torch.maximum(top, sink)
        top = top.masked_fill(top == -math.inf, 0.0)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        if st["sink"] is not None:
            total = total + torch.exp(sink - top)
        o = (e @ vs) / total.masked_fill(total == 0, 1.0)
        o = o.reshape(b, hk, t1 - t0, g, d).transpose(1, 2).reshape(b, t1 - t0, h, d)
        out[:, t0:t1] = o.to(out.dtype)
        lse[:, :, t0:t1] = (top + torch.log(total)).reshape(b, hk, t1 - t0, g)
    return out, lse


def _plain_backward(st, out, lse):
    c, hk = st["case"], st["case"]["hk"]
    b, m, h, d = st["q"].shape
    g, scale = h // hk, d ** -0.5
    dq = torch.empty_like(out)
    dk = torch.zeros(b, hk, c["n"], d, dtype=torch.float32, device=out.device)
    dv = dk if st["v"] is None else torch.zeros_like(dk)
    dsink = torch.zeros(h, dtype=torch.float32, device=out.device)
    for t0, t1, p0, p1, first, lo in _blocks(c):
        rows = _block_rows(st["q"], t0, t1, hk)
        up = _block_rows(st["dout"], t0, t1, hk)
        ks = _block_keys(st["k"], first, lo, p1 + 1)
        vs = ks if st["v"] is None else _block_keys(st["v"], first, lo, p1 + 1)
        big = lse[:, :, t0:t1].reshape(b, hk, -1, 1)
        p = torch.exp((rows @ ks.transpose(2, 3)) * scale - big)
        p = p.masked_fill(~_block_mask(st, c, p0, p1, first, lo), 0.0)
        dp = up @ vs.transpose(2, 3)
        # rows' sum of dout * out, in the form sum of P * dP (the same number before rounding)
        delta = (p * dp).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        x = (ds @ ks).reshape(b, hk, t1 - t0, g, d).transpose(1, 2).reshape(b, t1 - t0, h, d)
        dq[:, t0:t1] = x.to(dq.dtype)
        for acc, part in ((dk, ds.transpose(2, 3) @ rows), (dv, p.transpose(2, 3) @ up)):
            acc[:, :, :first] += part[:, :, :first]
            acc[:, :, lo:p1 + 1] += part[:, :, first:]
        if st["sink"] is not None:
            sink = st["sink"].detach().reshape(hk, 1, g).expand(hk, t1 - t0, g).reshape(1, hk, -1, 1)
            x = (torch.exp(sink - big) * delta).reshape(b, hk, t1 - t0, g)
            dsink -= x.sum((0, 2)).reshape(h)
    grads = [dq, dk.transpose(1, 2).to(dq.dtype)]
    if st["v"] is not None:
        grads.append(dv.transpose(1, 2).to(dq.dtype))
    if st["sink"] is not None:
        grads.append(dsink)
    return grads


def _slots(table, positions, page):
    """Slot numbers of positions [b, t] (or [t]) through the table."""
    b = table.shape[0]
    positions = positions.long().expand(b, -1)
    return table.long().gather(1, positions // page) * page + positions % page


def _decode(st):
    c = st["case"]
    # the call adds to the weights: a pass works on its own copy of the earlier ones
    weights = None if st["weights"] is None else st["weights"].clone()
    if own:
        from ascendc_kernel_b200.paged_cache import paged_attn
        out = paged_attn(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], st["sink"],
                         window=c["window"], n_first=c["first"], weights=weights)
        return out if weights is None else [out, weights]
    page, hk, d = c["page"], c["hk"], c["d"]
    g = c["h"] // hk
    pos = torch.arange(c["length"], device=st["q"].device)
    slots = _slots(st["table"], pos, page)
    out = torch.empty_like(st["q"])
    for i in range(c["b"]):
        ks = st["k_pages"].reshape(-1, hk, d)[slots[i]].float().transpose(0, 1)
        vs = ks
        if st["v_pages"] is not None:
            vs = st["v_pages"].reshape(-1, hk, d)[slots[i]].float().transpose(0, 1)
        vis = pos < st["lens"][i]
        if c["window"]:
            vis = vis & ((pos >= st["lens"][i] - c["window"]) | (pos < c["first"]))
        s = (st["q"][i].float().reshape(hk, g, d) * d ** -0.5) @ ks.transpose(1, 2)
        s = s.masked_fill(~vis, -math.inf)
        top = s.amax(-1, keepdim=True)
        if st["sink"] is not None:
            top = torch.maximum(top, st["sink"].reshape(hk, g, 1))
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        if st["sink"] is not None:
            total = total + torch.exp(st["sink"].reshape(hk, g, 1) - top)
        out[i] = ((e @ vs) / total).reshape(hk * g, d).to(out.dtype)
        if weights is not None:
            weights.view(-1)[slots[i]] += (e / total).sum((0, 1))
    return out if weights is None else [out, weights]


def _evict(st):
    c = st["case"]
    pools = [x for x in (st["k_pages"], st["v_pages"], st["weights"]) if x is not None]
    if own:
        from ascendc_kernel_b200.paged_cache import cache_evict
        kept, left = cache_evict(st["k_pages"], st["v_pages"], st["weights"], st["table"],
                                 st["lens"], st["dst"], budget=c["budget"], n_first=c["first"],
                                 n_recent=c["recent"])
        return [kept, left, *pools]
    page, budget = c["page"], c["budget"]
    pos = torch.arange(c["length"], device=st["weights"].device)
    slots = _slots(st["table"], pos, page)
    lens = st["lens"][:, None]
    rank = st["weights"].reshape(-1)[slots]
    rank = rank.masked_fill((pos < c["first"]) | (pos >= lens - c["recent"]), math.inf)
    rank = rank.masked_fill(pos >= lens, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]
    left = torch.clamp(lens, max=budget)
    valid = torch.arange(order.shape[1], device=pos.device) < left
    kept = torch.sort(order.masked_fill(~valid, c["length"]), dim=1).values
    if kept.shape[1] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[1]), value=c["length"])
    room = st["dst"].shape[1] * page
    spots = torch.arange(room, device=pos.device)
    valid = spots < left
    source = torch.nn.functional.pad(kept, (0, room - budget), value=0)
    source = slots.gather(1, source.masked_fill(~valid, 0))
    target = _slots(st["dst"], spots, page)
    for x in (st["k_pages"], st["v_pages"]):
        if x is not None:
            flat = x.view(-1, c["hk"], c["d"])
            flat[target] = torch.where(valid[..., None, None], flat[source], flat[target])
    flat = st["weights"].view(-1)
    flat[target] = torch.where(valid, flat[source], torch.zeros((), device=pos.device))
    kept = kept.masked_fill(kept == c["length"], -1).to(torch.int32)
    return [kept, left.reshape(-1).to(torch.int32), *pools]


def _append(st):
    c = st["case"]
    pools = [x for x in (st["k_pages"], st["v_pages"], st["weights"]) if x is not None]
    if own:
        from ascendc_kernel_b200.paged_cache import cache_append
        cache_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["start"],
                     weights=st["weights"])
        return pools
    pos = st["start"][:, None] + torch.arange(c["t"], device=st["k"].device)
    slots = _slots(st["table"], pos, c["page"])
    st["k_pages"].view(-1, c["hk"], c["d"])[slots] = st["k"]
    if st["v"] is not None:
        st["v_pages"].view(-1, c["hk"], c["d"])[slots] = st["v"]
    st["weights"].view(-1)[slots] = 0.0
    return pools


# ------------------------------------------------------------------ the definition in fp64
def exact(case, seed):
    if case["kind"] in ("evict", "append"):
        return None
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "decode":
            return _exact_decode(st)
        return _exact_window(st)


def _exact_window(st):
    """Head by head over whole score matrices."""
    c = st["case"]
    b, m, h, d = st["q"].shape
    n, hk = c["n"], c["hk"]
    dev = st["q"].device
    wide = torch.float64
    query = torch.arange(n - m, n, device=dev).unsqueeze(1)
    key = torch.arange(n, device=dev).unsqueeze(0)
    hidden = (key > query) | ((query - key >= c["window"]) & (key >= c["first"]))
    out = torch.zeros(b, m, h, d, dtype=wide, device=dev)
    train = c["kind"] == "train"
    if train:
        dq = torch.zeros_like(out)
        dk = torch.zeros(b, n, hk, d, dtype=wide, device=dev)
        dv = torch.zeros_like(dk)
        dsink = torch.zeros(h, dtype=wide, device=dev)
    values = st["k"] if st["v"] is None else st["v"]
    for i in range(b):
        mask = hidden if st["lens"] is None else hidden | (key >= st["lens"][i])
        for j in range(h):
            kk, vv = st["k"][i, :, j * hk // h].to(wide), values[i, :, j * hk // h].to(wide)
            qq = st["q"][i, :, j].to(wide)
            logit = (qq @ kk.T) / math.sqrt(d)
            logit[mask] = -math.inf
            if st["sink"] is not None:
                column = st["sink"][j].to(wide).expand(m, 1)
                prob = torch.softmax(torch.cat([logit, column], 1), 1)
                rest, prob = prob[:, n], prob[:, :n]
            else:
                prob = torch.nan_to_num(torch.softmax(logit, 1), nan=0.0)
            out[i, :, j] = prob @ vv
            if train:
                gg = st["dout"][i, :, j].to(wide)
                slope = gg @ vv.T
                mean = (gg * out[i, :, j]).sum(1, keepdim=True)
                slope = prob * (slope - mean)
                dq[i, :, j] = slope @ kk / math.sqrt(d)
                dk[i, :, j * hk // h] += slope.T @ qq / math.sqrt(d)
                dv[i, :, j * hk // h] += prob.T @ gg
                if st["sink"] is not None:
                    dsink[j] -= (rest * mean[:, 0]).sum()
    if not train:
        return out
    grads = [out, dq] + ([dk + dv] if st["v"] is None else [dk, dv])
    return grads + ([dsink] if st["sink"] is not None else [])


def _exact_decode(st):
    c = st["case"]
    wide = torch.float64
    hk, d, h = c["hk"], c["d"], c["h"]
    out = torch.zeros(c["b"], h, d, dtype=wide, device=st["q"].device)
    total = None if st["weights"] is None else st["weights"].to(wide)
    for i, length in enumerate(_lengths(c)):
        seen = list(range(length))
        if c["window"]:
            seen = [j for j in seen if j >= length - c["window"] or j < c["first"]]
        seen = torch.tensor(seen, device=out.device)
        at, row = st["table"][i].long()[seen // c["page"]], seen % c["page"]
        kk = st["k_pages"][at, row].to(wide)
        vv = kk if st["v_pages"] is None else st["v_pages"][at, row].to(wide)
        for j in range(hk):
            mine = slice(j * (h // hk), (j + 1) * (h // hk))
            logit = st["q"][i, mine].to(wide) @ kk[:, j].T / math.sqrt(d)
            if st["sink"] is not None:
                logit = torch.cat([logit, st["sink"][mine].to(wide).unsqueeze(1)], 1)
            prob = torch.softmax(logit, 1)[:, :len(seen)]
            out[i, mine] = prob @ vv[:, j]
            if total is not None:
                total[at, row] += prob.sum(0)
    return out if total is None else [out, total]

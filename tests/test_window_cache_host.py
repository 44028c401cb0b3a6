"""Host-side checks of the windowed-attention and paged-cache entry points: bad arguments
are refused before any CUDA work, empty calls are no-ops, workspace sizes are consistent;
the page accounting of PagedKVCache runs on the CPU with the GPU calls replaced."""

import ctypes

import pytest
import torch

from ascendc_kernel_b200 import _native, paged_cache

OK, INVALID, UNSUPPORTED, MISALIGNED, WORKSPACE = 0, 1, 2, 3, 5
FAKE = 0x1000  # 16-byte aligned, never dereferenced: every call below ends before a launch


def strides(*x):
    return (ctypes.c_int64 * len(x))(*x)


def fwd(**kw):
    a = dict(q=FAKE, qs=None, k=FAKE, ks=None, v=FAKE, vs=None, sink=None, lens=None, out=FAKE,
             lse=None, dtype=0, b=2, m=8, n=8, h=8, hk=2, d=64, w=4, f=0, scale=0.1)
    a.update(kw)
    return _native.lib().dsa_window_attn_fwd(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["sink"], a["lens"], a["out"], a["lse"],
        a["dtype"], a["b"], a["m"], a["n"], a["h"], a["hk"], a["d"], a["w"], a["f"], a["scale"], None)


WINDOW = [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(b=-1), INVALID), (dict(m=-1), INVALID), (dict(n=-1), INVALID), (dict(h=0), INVALID),
    (dict(hk=3), INVALID), (dict(w=0), INVALID), (dict(f=-1), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(dtype=2), UNSUPPORTED), (dict(d=96), UNSUPPORTED), (dict(h=129, hk=1), UNSUPPORTED),
    (dict(n=1 << 29), UNSUPPORTED), (dict(q=FAKE + 2), MISALIGNED), (dict(v=FAKE + 8), MISALIGNED),
    (dict(qs=strides(4096, 513, 64)), MISALIGNED), (dict(ks=strides(1024, 0, 64)), UNSUPPORTED),
    (dict(ks=strides(1024, -128, 64)), UNSUPPORTED), (dict(b=0), OK), (dict(m=0), OK),
    (dict(b=0, q=None, k=None, v=None, out=None), OK),
]


@pytest.mark.parametrize("kw,code", WINDOW + [(dict(out=None), INVALID),
                                              (dict(out=FAKE + 4), MISALIGNED)])
def test_window_forward_arguments(kw, code):
    assert fwd(**kw) == code


def bwd(**kw):
    a = dict(q=FAKE, qs=None, k=FAKE, ks=None, v=FAKE, vs=None, sink=None, lens=None, out=FAKE,
             lse=FAKE, dout=FAKE, dos=None, dq=FAKE, dk=FAKE, dv=FAKE, dsink=None, dtype=0, b=2, m=8,
             n=8, h=8, hk=2, d=64, w=4, f=0, scale=0.1, ws=FAKE, wb=1 << 40)
    a.update(kw)
    return _native.lib().dsa_window_attn_bwd(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["sink"], a["lens"], a["out"], a["lse"],
        a["dout"], a["dos"], a["dq"], a["dk"], a["dv"], a["dsink"], a["dtype"], a["b"], a["m"],
        a["n"], a["h"], a["hk"], a["d"], a["w"], a["f"], a["scale"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("kw,code", [x for x in WINDOW if "m" not in x[0] or x[0]["m"] != 0] + [
    (dict(out=None), INVALID), (dict(lse=None), INVALID), (dict(dout=None), INVALID),
    (dict(dq=None), INVALID), (dict(dk=None), INVALID), (dict(dsink=FAKE), INVALID),
    (dict(dv=None, v=FAKE + 16), INVALID),              # one gradient needs one tensor
    (dict(dout=FAKE + 4), MISALIGNED), (dict(dos=strides(4096, 512, 60)), MISALIGNED),
    (dict(ws=None), WORKSPACE), (dict(wb=100), WORKSPACE), (dict(ws=FAKE + 16), MISALIGNED),
])
def test_window_backward_arguments(kw, code):
    assert bwd(**kw) == code


def test_window_backward_workspace():
    f = _native.lib().dsa_window_attn_bwd_workspace_bytes
    assert f(2, 8, 8, 8, 3, 64, 4, 0, 0) == 0          # refused arguments
    one, two = f(1, 2600, 2600, 64, 1, 128, 128, 4, 1), f(2, 2600, 2600, 64, 1, 128, 128, 4, 1)
    assert 2600 * 64 * 12 < one < two
    assert f(1, 2600, 2600, 64, 1, 128, 128, 4, 0) > one  # two gradients of split key tiles


def dec(**kw):
    a = dict(q=FAKE, qs=None, k=FAKE, ks=None, v=FAKE, vs=None, table=FAKE, lens=FAKE, sink=None,
             out=FAKE, lse=None, w=None, dtype=0, b=2, h=8, hk=2, d=64, np=10, page=16, mp=4, win=0,
             f=0, scale=0.1, ws=FAKE, wb=1 << 40)
    a.update(kw)
    return _native.lib().dsa_paged_attn_fwd(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["table"], a["lens"], a["sink"],
        a["out"], a["lse"], a["w"], a["dtype"], a["b"], a["h"], a["hk"], a["d"], a["np"], a["page"],
        a["mp"], a["win"], a["f"], a["scale"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(table=None), INVALID), (dict(lens=None), INVALID), (dict(out=None), INVALID),
    (dict(b=-1), INVALID), (dict(h=7), INVALID), (dict(np=0), INVALID), (dict(mp=0), INVALID),
    (dict(win=-1), INVALID), (dict(f=-1), INVALID), (dict(scale=-1.0), INVALID),
    (dict(dtype=5), UNSUPPORTED), (dict(d=256), UNSUPPORTED), (dict(page=12), UNSUPPORTED),
    (dict(h=258), UNSUPPORTED), (dict(mp=1 << 26), UNSUPPORTED), (dict(b=70000), UNSUPPORTED),
    (dict(q=FAKE + 8), MISALIGNED), (dict(ws=None), WORKSPACE), (dict(wb=64), WORKSPACE),
    (dict(ws=FAKE + 16), MISALIGNED), (dict(b=0), OK),
])
def test_paged_attention_arguments(kw, code):
    assert dec(**kw) == code


def app(**kw):
    a = dict(k=FAKE, ks=None, v=FAKE, vs=None, kp=FAKE, kps=None, vp=FAKE, vps=None, w=None,
             table=FAKE, start=FAKE, b=2, t=3, hk=2, d=64, np=10, page=16, mp=4)
    a.update(kw)
    return _native.lib().dsa_cache_append(
        a["k"], a["ks"], a["v"], a["vs"], a["kp"], a["kps"], a["vp"], a["vps"], a["w"], a["table"],
        a["start"], a["b"], a["t"], a["hk"], a["d"], a["np"], a["page"], a["mp"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), INVALID), (dict(kp=None), INVALID), (dict(v=None), INVALID),
    (dict(vp=None), INVALID), (dict(start=None), INVALID), (dict(t=-1), INVALID),
    (dict(page=0), INVALID), (dict(d=60), UNSUPPORTED), (dict(k=FAKE + 4), MISALIGNED),
    (dict(kp=FAKE + 4), MISALIGNED), (dict(ks=strides(384, 127, 64)), MISALIGNED),
    (dict(kps=strides(-8, 128, 64)), UNSUPPORTED), (dict(b=0), OK), (dict(t=0), OK),
])
def test_append_arguments(kw, code):
    assert app(**kw) == code


def evi(**kw):
    a = dict(kp=FAKE, kps=None, vp=FAKE, vps=None, w=FAKE, table=FAKE, lens=FAKE, dst=FAKE,
             kept=FAKE, left=FAKE, b=2, hk=2, d=64, np=10, page=16, mp=4, dp=2, budget=20, f=4, r=4)
    a.update(kw)
    return _native.lib().dsa_cache_evict(
        a["kp"], a["kps"], a["vp"], a["vps"], a["w"], a["table"], a["lens"], a["dst"], a["kept"],
        a["left"], a["b"], a["hk"], a["d"], a["np"], a["page"], a["mp"], a["dp"], a["budget"],
        a["f"], a["r"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(kp=None), INVALID), (dict(w=None), INVALID), (dict(table=None), INVALID),
    (dict(lens=None), INVALID), (dict(dst=None), INVALID), (dict(kept=None), INVALID),
    (dict(left=None), INVALID), (dict(budget=0), INVALID), (dict(f=17), INVALID),
    (dict(r=-1), INVALID), (dict(budget=33), INVALID), (dict(dp=0), INVALID),
    (dict(d=12), UNSUPPORTED), (dict(b=65536), UNSUPPORTED), (dict(kp=FAKE + 2), MISALIGNED),
    (dict(b=0), OK),
])
def test_evict_arguments(kw, code):
    assert evi(**kw) == code


def test_page_accounting_on_the_host(monkeypatch):
    seen = []

    def append(k, v, kp, vp, table, start, weights):
        seen.append((table.clone(), start.clone()))

    def evict(kp, vp, weights, table, lens, dst, *, budget, n_first, n_recent):
        return None, torch.clamp(lens, max=budget)

    monkeypatch.setattr(paged_cache, "cache_append", append)
    monkeypatch.setattr(paged_cache, "cache_evict", evict)
    c = paged_cache.PagedKVCache(2, 9, 8, 40, 1, 64, track_weights=True, device="cpu")
    c.append(torch.zeros(2, 9, 1, 64))
    assert c.pages == [[0, 1], [2, 3]] and c.lens.tolist() == [9, 9]
    assert seen[-1][0].tolist() == [[0, 1, -1, -1, -1], [2, 3, -1, -1, -1]]
    c.append(torch.zeros(2, 7, 1, 64))           # fills the pages: none is taken
    assert len(c.free) == 5 and seen[-1][1].tolist() == [9, 9]
    c.evict(4)                                   # one fresh page each, the old ones are free
    assert c.host_lens == [4, 4] and c.lens.tolist() == [4, 4]
    assert sorted(c.free + c.pages[0] + c.pages[1]) == list(range(9))
    assert not set(c.pages[0]) & {0, 1, 2, 3} and len(c.pages[0]) == 1
    c.evict(30)                                  # nothing to drop: still moved, pages balanced
    assert c.host_lens == [4, 4] and sorted(c.free + c.pages[0] + c.pages[1]) == list(range(9))
    with pytest.raises(RuntimeError, match="exhausted"):
        c.append(torch.zeros(2, 36, 1, 64))
    assert c.host_lens == [4, 4] and sorted(c.free + c.pages[0] + c.pages[1]) == list(range(9))
    with pytest.raises(AssertionError):
        c.append(torch.zeros(2, 37, 1, 64))

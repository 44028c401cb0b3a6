"""fp16 windowed and paged attention with the bounds that its arithmetic gives.

u = 2^-11 is the unit roundoff of fp16; below 2^-14 its step is 2^-24, so a rounding is off by
2^-25 at most there. Forward: a weight P is rounded relative to a reference that is a score
already seen, never above the row's maximum, so the divisor is at least 1 and, divided by it, a
subnormal weight is off by at most 2^-25 a key; P of normal size by u P; the output by its own
rounding. The fp32 part is 1e-4 of the magnitudes (scores below 30 are good to 2e-5).

Backward: P <= 1 is rounded as 2^14 P: 2^-39 a key. dS = P (dP - D) is rounded in units of
B 2^-14, where B is a power of two at most twice above |dout| |v| + |D| (the largest row of
dout with this key, or the largest key with this row): off by 2^-38 (|dout| |v| + |D|). D comes
from the rounded out. The results carry their own rounding.
"""

import math

import pytest
import torch

from ascendc_kernel_b200 import _native
from ascendc_kernel_b200.paged_cache import paged_attn
from ascendc_kernel_b200.window_attn import window_attn, window_attn_bwd
from tests import test_paged_cache_gpu as paged_tests
from tests import test_window_attn_gpu as window_tests

pytestmark = pytest.mark.gpu

U, STEP, F32 = 2.0 ** -11, 2.0 ** -25, 1e-4


def definition(q, k, v, window, n_first, scale, dout):
    """fp64 values of out, dq, dk, dv with their bounds; q and dout [m, h, d], k and v
    [n, hk, d]."""
    (m, h, d), (n, hk) = q.shape, k.shape[:2]
    q, k, v, g = (x.double().transpose(0, 1) for x in (q, k, v, dout))
    k, v = k.repeat_interleave(h // hk, 0), v.repeat_interleave(h // hk, 0)
    pos = torch.arange(m, device=q.device)[:, None] + n - m
    j = torch.arange(n, device=q.device)[None]
    see = (j <= pos) & ((j > pos - window) | (j < n_first))
    p = torch.softmax((q @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf), -1)
    see = see.double()
    r, e = {}, {}
    r["out"] = p @ v
    mag = p @ v.abs()
    e["out"] = U * (r["out"].abs() + mag) + F32 * mag + STEP * (see @ v.abs()) + STEP
    dp = g @ v.transpose(1, 2)
    delta = (g * r["out"]).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (g.abs() * e["out"]).sum(-1, keepdim=True)
    unit = g.norm(dim=-1).max() * v.norm(dim=-1).max() + (delta.abs() + e_delta).max()
    e_ds = U * ds.abs() + (1 + U) * p * e_delta + F32 * p * (dp.abs() + delta.abs()) \
        + 2.0 ** -38 * unit * see
    e_p = (U + F32) * p + 2.0 ** -39 * see

    def group(x):
        return x.reshape(hk, h // hk, n, d).sum(1)

    r["dq"], e["dq"] = ds @ k * scale, e_ds @ k.abs() * scale
    r["dk"] = group(ds.transpose(1, 2) @ q * scale)
    e["dk"] = group(e_ds.transpose(1, 2) @ q.abs() * scale)
    r["dv"], e["dv"] = group(p.transpose(1, 2) @ g), group(e_p.transpose(1, 2) @ g.abs())
    for x in ("dq", "dk", "dv"):
        e[x] = e[x] + U * r[x].abs() + STEP
    # the bounds are of first order in u
    return ({x: y.transpose(0, 1) for x, y in r.items()},
            {x: (1 + 2.0 ** -4) * y.transpose(0, 1) for x, y in e.items()})


def within(got, want, bound, what):
    """`got` keeps to the bound, and a result of zeros would not."""
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs() > bound
    assert not off.any(), (what, off.float().mean().item())
    assert (want.abs() > bound).float().mean() > 0.5, what + ": the bound says nothing"


# m, n, h, hk, window, n_first: many keys to a row; a window; a group above 64
@pytest.mark.parametrize("m,n,h,hk,window,first", [
    (900, 900, 4, 2, 900, 0), (700, 1100, 6, 1, 257, 5), (130, 400, 77, 1, 400, 0)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e-5, 1e-3, 1.0, 3000.0])
def test_gradients_of_small_and_large_upstream(cuda_device, m, n, h, hk, window, first, d, size):
    g = torch.Generator(device="cuda").manual_seed(11)

    def r(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q, k, v = (r(*x).half() for x in ((m, h, d), (n, hk, d), (n, hk, d)))
    dout = (r(m, h, d) * size).half()
    want, bound = definition(q, k, v, window, first, d ** -0.5, dout)
    assert max(want[x].abs().max() for x in ("dq", "dk", "dv")) < 60000, "fp16 holds the result"
    out, lse = window_attn(q[None], k[None], v[None], window=window, n_first=first,
                           return_lse=True)
    within(out[0], want["out"], bound["out"], "out")
    got = window_attn_bwd(dout[None], q[None], k[None], v[None], None, out, lse, window=window,
                          n_first=first)
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x[0], want[name], bound[name], name)
    # K and V one tensor: dk receives both
    want, bound = definition(q, k, k, window, first, d ** -0.5, dout)
    out, lse = window_attn(q[None], k[None], window=window, n_first=first, return_lse=True)
    dq, dk, dv, _ = window_attn_bwd(dout[None], q[None], k[None], None, None, out, lse,
                                    window=window, n_first=first)
    assert dv is None
    within(dq[0], want["dq"], bound["dq"], "dq")
    within(dk[0], want["dk"] + want["dv"], bound["dk"] + bound["dv"], "dk + dv")
    assert _native.device_error(0) == 0


@pytest.mark.parametrize("d", [64, 128])
def test_gradients_where_ds_passes_fp16(cuda_device, d):
    """dS beyond 65504 with gradients well below it: values of +-1 under an upstream gradient
    that lines up with them, small keys and queries."""
    m, h, size = 300, 2, 4000.0
    g = torch.Generator(device="cuda").manual_seed(13)

    def r(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    sign = torch.where(r(d) > 0, 1.0, -1.0)
    q, k = (r(m, h, d) * 0.25).half(), (r(m, 1, d) * 0.25).half()
    v = (sign * torch.where(torch.arange(m, device="cuda") % 2 > 0, 1.0, -1.0)[:, None])[:, None].half()
    dout = (sign * size * torch.where(r(m, h, 1) > 0, 1.0, -1.0)).half()
    want, bound = definition(q, k, v, m, 0, d ** -0.5, dout)
    p0 = torch.softmax((k[:2, 0].double() @ q[1, 0].double()) * d ** -0.5, 0)
    assert 2 * p0[0] * p0[1] * size * d > 65504, "dS of the second row's first key"
    assert max(want[x].abs().max() for x in ("dq", "dk", "dv")) < 60000, "fp16 holds the result"
    out, lse = window_attn(q[None], k[None], v[None], window=m, return_lse=True)
    got = window_attn_bwd(dout[None], q[None], k[None], v[None], None, out, lse, window=m)
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x[0], want[name], bound[name], name)
    assert _native.device_error(0) == 0


@pytest.mark.parametrize("rows,h,hk,d", [(5000, 8, 2, 64), (9000, 64, 1, 128), (30000, 8, 2, 64),
                                         (30000, 128, 1, 64)])
def test_long_paged_rows(cuda_device, rows, h, hk, d):
    page = 64
    g = torch.Generator(device="cuda").manual_seed(3)
    width = -(-rows // page)
    k = torch.randn(width, page, hk, d, generator=g, device="cuda").half()
    v = torch.randn(width, page, hk, d, generator=g, device="cuda").half()
    q = torch.randn(1, h, d, generator=g, device="cuda").half()
    table = torch.arange(width, dtype=torch.int32, device="cuda")[None].contiguous()
    n = torch.full((1,), rows, dtype=torch.int32, device="cuda")
    out = paged_attn(q, k, v, table, n)
    kk, vv = (x.reshape(-1, hk, d)[:rows].double().transpose(0, 1).repeat_interleave(h // hk, 0)
              for x in (k, v))
    p = torch.softmax((kk @ q[0].double()[:, :, None])[..., 0] * d ** -0.5, -1)[:, None]
    want, mag = (p @ vv)[:, 0], (p @ vv.abs())[:, 0]
    bound = U * (want.abs() + mag) + F32 * mag + STEP * (vv.abs().sum(1) + 1)
    within(out[0], want, bound, "out")
    assert _native.device_error(0) == 0


@pytest.fixture
def step(monkeypatch):
    """The other files' bounds with 2^-25 a key for fp16 in place of their 2^-17: where their
    reference lies 2^8 below the maximum, the divisor is that much larger too, and the
    gradients' P and dS are scaled. In the long cases 2^-17 a key allows anything."""
    monkeypatch.setitem(window_tests.TINY, torch.float16, STEP)
    monkeypatch.setitem(paged_tests.TINY, torch.float16, STEP)


@pytest.mark.parametrize("shape", window_tests.SHAPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sink,shared,ragged", [(True, True, False), (False, False, True),
                                                (True, False, True), (False, True, False)])
def test_window_shapes(cuda_device, step, shape, d, sink, shared, ragged):
    window_tests.test_forward_and_gradients(cuda_device, shape, d, torch.float16, sink, shared,
                                            ragged)


def test_window_score_range(cuda_device, step):
    window_tests.test_large_and_small_scores(cuda_device)


@pytest.mark.parametrize("case", paged_tests.CASES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sink,shared", [(True, True), (False, False)])
def test_paged_cases(cuda_device, step, case, d, sink, shared):
    paged_tests.test_paged_attention(cuda_device, case, d, torch.float16, sink, shared)

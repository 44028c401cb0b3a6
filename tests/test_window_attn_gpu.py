"""Windowed attention (forward and backward) against its definition in fp64.

Bounds. With u the unit roundoff of the operands' type (2^-8 bf16, 2^-11 fp16), an output
carries its own rounding (u |out|) and that of the weights P before the second product
(u sum P |v|). The scores are fp32 sums of exact products: at head_dim <= 128 and |q| |k|
scale <= 30 their error is below 2e-5, exp and the sums add less, so the fp32 part is
bounded by 1e-4 of the sum of magnitudes. fp16 weights below 2^-14 are subnormal with an
absolute step of 2^-24: half of it a key, against weights that are up to 2^8 away from the
largest. The gradients sum products of P or dS = P (dP - D), rounded to the same type; D
comes from the rounded out, an error of u sum_d |dout| (|out| + sum P |v|).
"""

import math

import pytest
import torch

from ascendc_kernel_b200 import _native
from ascendc_kernel_b200.window_attn import WindowAttention, window_attn, window_attn_bwd

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -17}  # 2^-25 times the 2^8 of the reference
F32 = 1e-4


def definition(q, k, v, sink, window, n_first, lens, scale, dout=None):
    """Everything in fp64 over [b, h, m, n], with the sums of magnitudes the bounds need."""
    q, k, v = q.double(), k.double(), (k if v is None else v).double()
    b, m, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    kk, vv = (x.repeat_interleave(h // hk, 2).transpose(1, 2) for x in (k, v))
    qq = q.transpose(1, 2)
    pos = torch.arange(m, device=q.device)[:, None] + n - m
    j = torch.arange(n, device=q.device)[None]
    see = (j <= pos) & ((j > pos - window) | (j < n_first))
    see = see[None].expand(b, m, n)
    if lens is not None:
        see = see & (j[None] < lens[:, None, None])
    see = see[:, None]
    # hidden rows may hold anything: they are left out, not multiplied by 0
    if lens is not None:
        live = (torch.arange(n, device=q.device)[None] < lens[:, None])[:, None, :, None]
        kk, vv = torch.where(live, kk, 0.0), torch.where(live, vv, 0.0)
    s = (qq @ kk.transpose(2, 3) * scale).masked_fill(~see, -math.inf)
    col = None
    if sink is not None:
        col = sink.double()[None, :, None, None].expand(b, h, m, 1)
        s2 = torch.cat([s, col], -1)
    else:
        s2 = s
    lse = torch.logsumexp(s2, -1, keepdim=True)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)).masked_fill(~see, 0.0)
    r = {"out": (p @ vv).transpose(1, 2), "lse": lse[..., 0].transpose(1, 2)}
    r["out_mag"] = (p @ vv.abs()).transpose(1, 2)
    r["out_keys"] = (see.double() @ vv.abs()).expand(b, h, m, d).transpose(1, 2)
    if dout is None:
        return r
    g = dout.double().transpose(1, 2)
    o, mag = r["out"].transpose(1, 2), r["out_mag"].transpose(1, 2)
    dp = g @ vv.transpose(2, 3)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)

    def group(x):  # sum over the heads of a group, [b, hk, n, d] -> [b, n, hk, d]
        return x.reshape(b, hk, h // hk, *x.shape[2:]).sum(2).transpose(1, 2)

    r["dq"] = (ds @ kk * scale).transpose(1, 2)
    r["dk"] = group(ds.transpose(2, 3) @ qq * scale)
    r["dv"] = group(p.transpose(2, 3) @ g)
    u, tiny = U[dout.dtype], TINY[dout.dtype]
    # error of dS: its rounding, that of D, and fp32; one subnormal step
    d_err = (g.abs() * (u * o.abs() + u * mag + F32 * mag)).sum(-1, keepdim=True)
    e_ds = u * ds.abs() + p * d_err * (1 + u) + F32 * p * (dp.abs() + delta.abs()) \
        + tiny * see.double() * (1 + dp.abs())
    e_p = u * p + F32 * p + tiny * see.double()
    r["dq_err"] = (e_ds @ kk.abs() * scale).transpose(1, 2) + u * r["dq"].abs() + tiny
    r["dk_err"] = group(e_ds.transpose(2, 3) @ qq.abs() * scale) + u * r["dk"].abs() + tiny
    r["dv_err"] = group(e_p.transpose(2, 3) @ g.abs()) + u * r["dv"].abs() + tiny
    if sink is not None:
        ps = torch.exp(col - lse)
        r["dsink"] = -(ps[..., 0] * delta[..., 0]).sum((0, 2))
        r["dsink_err"] = F32 * (ps[..., 0] * (p * dp.abs()).sum(-1)).sum((0, 2))
    return r


def inputs(b, m, n, h, hk, d, dtype, sink, shared, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    return (r(b, m, h, d), r(b, n, hk, d), None if shared else r(b, n, hk, d),
            torch.randn(h, generator=g, device="cuda") * 2 if sink else None, r(b, m, h, d))


def check_out(out, r, dtype):
    bound = U[dtype] * (r["out"].abs() + r["out_mag"]) + F32 * r["out_mag"] \
        + TINY[dtype] * r["out_keys"] + TINY[dtype]
    assert torch.isfinite(out).all()
    assert ((out.double() - r["out"]).abs() <= bound).all()


# b, m, n, h, hk, window, n_first: one token; one head; short rows; a group that does not
# divide the tile; chunked prompts; windows across, at and beside the 32- and 128-key
# borders; first tokens beyond the window; a group of 128 and an odd one above 64; more
# queries than keys (empty rows); no key at all
SHAPES = [
    (1, 1, 1, 1, 1, 1, 0), (2, 5, 5, 16, 1, 3, 1), (2, 37, 37, 64, 1, 16, 4),
    (1, 300, 300, 4, 4, 128, 0), (2, 97, 300, 24, 8, 100, 7), (1, 130, 130, 128, 1, 500, 0),
    (2, 65, 411, 12, 2, 200, 130), (2, 100, 60, 8, 2, 20, 2), (1, 400, 400, 1, 1, 128, 200),
    (2, 64, 64, 14, 2, 9, 0), (1, 70, 90, 77, 1, 50, 3), (1, 257, 257, 2, 1, 129, 33),
    (1, 1, 385, 8, 1, 127, 32), (2, 7, 0, 4, 2, 5, 2),
    # ragged: the second tile's window starts past the valid keys
    (1, 540, 540, 1, 1, 20, 0), (1, 540, 540, 1, 1, 20, 5),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.bfloat16),
                                     (128, torch.float16), (64, torch.float16)])
@pytest.mark.parametrize("sink,shared,ragged", [(True, True, False), (False, False, True),
                                                (True, False, True), (False, True, False)])
def test_forward_and_gradients(cuda_device, shape, d, dtype, sink, shared, ragged):
    b, m, n, h, hk, window, first = shape
    q, k, v, s, dout = inputs(b, m, n, h, hk, d, dtype, sink, shared)
    lens = None
    if ragged:
        # a whole, a partial and an empty sequence; rows past a length hold NaN and Inf
        lens = torch.tensor([n * 2 // 3, 0, n][:b], dtype=torch.int32, device="cuda")
        for i in range(b):
            for x in (k, v):
                if x is not None:
                    x[i, lens[i]:] = math.nan
                    x[i, lens[i]::2] = math.inf
    scale = d ** -0.5
    r = definition(q, k, v, s, window, first, lens, scale, dout)
    kw = dict(window=window, n_first=first, kv_lens=lens)
    out, lse = window_attn(q, k, v, s, return_lse=True, **kw)
    check_out(out, r, dtype)
    dead = r["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, dead)
    assert ((lse.double() - r["lse"])[~dead].abs() <= F32 * (1 + r["lse"][~dead].abs())).all()
    got = window_attn_bwd(dout, q, k, v, s, out, lse, **kw)
    again = window_attn_bwd(dout, q, k, v, s, out, lse, **kw)
    want = dict(r, dk=r["dk"] + r["dv"], dk_err=r["dk_err"] + r["dv_err"]) if shared else r
    for name, x, y in zip(("dq", "dk", "dv", "dsink"), got, again):
        if x is None:
            assert name == ("dv" if shared else "dsink") or (name == "dsink" and not sink)
            continue
        assert torch.equal(x, y), name + " is deterministic"
        assert torch.isfinite(x).all(), name
        err = (x.double() - want[name]).abs()
        # the bounds are of first order in u; the rest is below a sixteenth of them
        assert (err <= (1 + 2.0 ** -4) * want[name + "_err"] + 1e-30).all(), name
    assert _native.device_error(0) == 0


def test_key_tiles_split_over_their_rows(cuda_device):
    """One kv head under 64 query heads: few key tiles, split and joined; the first tokens'
    tile is seen by every row."""
    b, m, h, d, dtype = 1, 700, 64, 128, torch.bfloat16
    q, k, v, s, dout = inputs(b, m, m, h, 1, d, dtype, True, False)
    r = definition(q, k, v, s, 64, 4, None, d ** -0.5, dout)
    out, lse = window_attn(q, k, v, s, window=64, n_first=4, return_lse=True)
    check_out(out, r, dtype)
    got = window_attn_bwd(dout, q, k, v, s, out, lse, window=64, n_first=4)
    for name, x in zip(("dq", "dk", "dv", "dsink"), got):
        assert ((x.double() - r[name]).abs() <= (1 + 2.0 ** -4) * r[name + "_err"]).all(), name



@pytest.mark.parametrize("lens", [[204, 0, 0], [0, 0, 0], [0, 204, 0]])
def test_long_runs_of_rows_without_keys(cuda_device, lens):
    """Several work items in a row on each SM see no key, after and before some that do."""
    q, k, v, s, _ = inputs(3, 153, 204, 381, 3, 64, torch.bfloat16, True, False)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    _native.device_error(0)
    out = window_attn(q, k, v, s, window=2, n_first=65, kv_lens=n)
    assert _native.device_error(0) == 0
    check_out(out, definition(q, k, v, s, 2, 65, n, 64 ** -0.5), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_against_differences(cuda_device, dtype):
    """The directional derivative of sum(out * dout) from the gradients, against a central
    difference of the fp64 definition."""
    b, m, h, hk, d = 1, 50, 6, 2, 64
    q, k, v, s, dout = inputs(b, m, m, h, hk, d, dtype, True, False)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, s)]
    out = window_attn(*leaves, window=17, n_first=3)
    grads = torch.autograd.grad(out, leaves, dout)
    r = definition(q, k, v, s, 17, 3, None, d ** -0.5, dout)
    g = torch.Generator(device="cuda").manual_seed(5)
    eps = 1e-5
    for i, (x, dx, name) in enumerate(zip((q, k, v, s), grads, ("dq", "dk", "dv", "dsink"))):
        step = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)
        value = []
        for sign in (1, -1):
            args = [y.double() for y in (q, k, v, s)]
            args[i] = args[i] + sign * eps * step
            o = definition(*args, 17, 3, None, d ** -0.5)["out"]
            value.append((o * dout.double()).sum())
        slope = (value[0] - value[1]) / (2 * eps)
        mine = (dx.double() * step).sum()
        bound = ((1 + 2.0 ** -4) * r[name + "_err"] * step.abs()).sum()
        assert abs(mine - slope) <= bound + 1e-6 * abs(slope)


def test_large_and_small_scores(cuda_device):
    """Scores that climb by hundreds along the keys move the running reference; a sink far
    above and far below them neither overflows nor loses the row."""
    b, m, h, d = 1, 300, 2, 64
    q = torch.zeros(b, m, h, d, device="cuda", dtype=torch.float16)
    q[..., 0] = 8.0
    k = torch.randn(b, m, 1, d, device="cuda").half() * 0.1
    k[0, :, 0, 0] = torch.linspace(-100, 100, m, device="cuda").half()
    v = torch.randn(b, m, 1, d, device="cuda").half()
    for level in (-1000.0, 0.0, 90.0, 1000.0, -math.inf):
        s = torch.full((h,), level, device="cuda")
        r = definition(q, k, v, s, 200, 4, None, d ** -0.5)
        out, lse = window_attn(q, k, v, s, window=200, n_first=4, return_lse=True)
        # scores of 100: their fp32 error grows with them (2^-22 |s|, twice)
        bound = (2.0 ** -11 + 2.0 ** -13) * (r["out"].abs() + r["out_mag"]) \
            + TINY[torch.float16] * (1 + r["out_keys"])
        assert ((out.double() - r["out"]).abs() <= bound).all()
        assert ((lse.double() - r["lse"]).abs() <= F32 * (1 + r["lse"].abs())).all()


def test_strides_streams_and_module(cuda_device):
    """Operands as views of fused and transposed buffers, on another stream than the one
    they were made on, through the module and autograd."""
    b, m, h, hk, d = 2, 150, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(b, m, h + 2 * hk, d, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)      # [b, h, m, d] in memory
    odd = torch.randn(b, m, h, d + 1, generator=g, device="cuda").to(torch.bfloat16)[..., 1:]
    layer = WindowAttention(h, d, window=40, n_first=3).cuda()
    torch.nn.init.normal_(layer.attn_sink)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = window_attn(q.contiguous(), k.contiguous(), v.contiguous(), layer.attn_sink.detach(),
                       window=40, n_first=3)
    with torch.cuda.stream(side):
        assert torch.equal(layer(q, k, v).detach(), want)
        assert torch.equal(layer(qt, k, v).detach(), want)
        a = window_attn(odd, k, v, window=40)
        assert torch.equal(a, window_attn(odd.contiguous(), k, v, window=40))
        leaf = qkv.clone().requires_grad_(True)
        out = layer(leaf[:, :, :h], leaf[:, :, h:h + hk], leaf[:, :, h + hk:])
        out.transpose(1, 2).float().sum().backward()         # a strided upstream gradient
        # an expanded upstream gradient (stride 0)
        (g2,) = torch.autograd.grad(layer(leaf[:, :, :h], k, v).sum(), leaf)
    torch.cuda.synchronize()
    ones = torch.ones_like(want)
    r = definition(q, k, v, layer.attn_sink.detach(), 40, 3, None, d ** -0.5, ones)
    got = leaf.grad.double()
    for name, x in (("dq", got[:, :, :h]), ("dk", got[:, :, h:h + hk]), ("dv", got[:, :, h + hk:])):
        assert ((x - r[name]).abs() <= (1 + 2.0 ** -4) * r[name + "_err"]).all(), name
    assert torch.equal(g2[:, :, :h], leaf.grad[:, :, :h])
    x = layer.attn_sink.grad.double()
    assert ((x - r["dsink"]).abs() <= r["dsink_err"]).all()


def test_offsets_past_32_bits(cuda_device):
    """A batch stride above 2^32 bytes."""
    b, m, d = 2, 40, 64
    far = 2 ** 31 + 512  # elements
    pool = torch.empty(far + m * d, dtype=torch.bfloat16, device="cuda")
    x = pool.as_strided((b, m, 1, d), (far, d, d, 1))
    x.copy_(torch.randn(b, m, 1, d, device="cuda"))
    y = x.clone()
    assert torch.equal(window_attn(x, x, window=9), window_attn(y, y, window=9))
    lse = window_attn(y, y, window=9, return_lse=True)
    for a, c in zip(window_attn_bwd(x, x, x, x, None, *lse, window=9)[:3],
                    window_attn_bwd(y, y, y, y, None, *lse, window=9)[:3]):
        assert torch.equal(a, c)


def test_empty_calls(cuda_device):
    for b, m, n in ((0, 4, 4), (2, 0, 4), (2, 0, 0)):
        q = torch.zeros(b, m, 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        k = torch.zeros(b, n, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        s = torch.zeros(4, device="cuda", requires_grad=True)
        out = window_attn(q, k, None, s, window=3)
        assert out.shape == q.shape
        dq, dk, ds = torch.autograd.grad(out.sum(), (q, k, s))
        assert not dk.any() and not ds.any() and dq.shape == q.shape


def test_refusals(cuda_device):
    q = torch.zeros(1, 8, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(1, 8, 2, 64, device="cuda", dtype=torch.bfloat16)
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = [
        dict(q=q.float()), dict(q=q.cpu()), dict(k=k.half()), dict(q=q[..., :32], k=k[..., :32]),
        dict(q=q[:, :, :3]), dict(v=k[:, :4]), dict(window=0), dict(n_first=-1),
        dict(softmax_scale=0.0), dict(kv_lens=lens.long()), dict(kv_lens=lens.cpu()),
        dict(sink=torch.zeros(3, device="cuda")), dict(out=q[..., ::2]), dict(out=q.half()),
    ]
    for kw in bad:
        a = dict(q=q, k=k, v=None, sink=None, window=4)
        a.update(kw)
        with pytest.raises(AssertionError):
            window_attn(**a)
    wide = torch.zeros(1, 8, 129, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        window_attn(wide, k[:, :, :1], window=4)
    with pytest.raises(AssertionError):
        window_attn(q.requires_grad_(True), k, window=4, out=torch.empty_like(q))

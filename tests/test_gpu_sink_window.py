"""Attention over a causal window with sinks (esa_sink_window_*) against
float64 (GPU).

Tolerances, with u = finfo(dtype).eps / 2 (0 in the products of float32) and
e = 2^-24.  A score is a float32 sum of D products, scaled and shifted:
E = (D + 8) e max(scale sum |q||k|) + 16 e (the exponential's own error among
them).  A probability is off by the factor E and, entering a product, by u; the
rows' normaliser is the sum of the probabilities that the product used, off by
the same.  So with n the keys of a row
  |o - ref|  <= (2 u + 2 E + n e) sum p |v| + u |ref|
  |lse - ref| <= E + (n + 8) e + 4 e |ref|
and in the backward, P being off by E and lse's error, delta by the error of o
times |dO|, dP by D e sum |dO||v|:
  |dS| is off by p (dP's + delta's) + (factor + u) p (|dP| + |delta|),
  dV by (factor + u + n e) P^T |dO|, dQ and dK by the sums of dS's with |k| and
  |q|, n e of their size each; every gradient by u of itself.
"""
import math

import pytest
import torch

from elastic_sparse_attention import ElasticSparseAttention
from layer_oracle import window_attention, window_mask
from qk_norm_rope import QKNormRope
from sink_window_attention import (SinkWindowAttention, sink_window_attention_bwd,
                                   sink_window_attention_fwd)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E24 = 2.0 ** -24


def rows(B, heads, n, D, dtype, gen, strided):
    if strided:
        return torch.randn(B, n, heads, D, generator=gen).to(dtype).transpose(1, 2)
    return torch.randn(B, heads, n, D, generator=gen).to(dtype)


def to_dev(t):
    """t on the device, in t's memory order."""
    if t.stride(1) < t.stride(2):
        return t.transpose(1, 2).to(DEV).transpose(1, 2)
    return t.to(DEV)


def units(dtype):
    u = torch.finfo(dtype).eps / 2
    return u, (0.0 if dtype == F32 else u)


def bounds(q, k, v, seen, scale, dtype, dout=None):
    """(reference results, their tolerances) as above."""
    u, up = units(dtype)
    D, G = q.shape[-1], q.shape[1] // k.shape[1]
    res = window_attention(q, k, v, seen, scale, dout)
    big = float((q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * scale)
    E = (D + 8) * E24 * big + 16 * E24
    n = seen.sum(-1).double()[:, None, :, None]  # [B, 1, Lq, 1]
    size, _ = window_attention(q, k, v.abs(), seen, scale)
    tol_o = (2 * up + 2 * E + n * E24) * size + u * res[0].abs()
    lse = res[1]
    tol_lse = E + (n[..., 0] + 8) * E24 + 4 * E24 * torch.where(torch.isinf(lse), 0.0, lse.abs())
    if dout is None:
        return res, (tol_o, tol_lse)
    B, H = q.shape[:2]
    kk, vv = (t.double().repeat_interleave(G, 1) for t in (k, v))
    qq, gg = q.double(), dout.double()
    vis = seen[:, None]
    s = torch.where(vis, qq @ kk.transpose(2, 3) * scale, -math.inf)
    p = torch.where(vis & torch.isfinite(lse)[..., None], torch.exp(s - lse[..., None]), 0.0)
    dp = gg @ vv.transpose(2, 3)
    delta = (gg * res[0]).sum(-1, keepdim=True)
    err_dp = D * E24 * (gg.abs() @ vv.abs().transpose(2, 3))
    err_delta = (gg.abs() * tol_o).sum(-1, keepdim=True) + D * E24 * (gg * res[0]).abs().sum(
        -1, keepdim=True)
    factor = E + tol_lse[..., None] + 8 * E24
    mag = p * (dp.abs() + delta.abs())
    err_ds = p * (err_dp + err_delta) + (factor + up) * mag
    nk = seen.sum(-2).double().max() * G + 64   # terms of a key's sums, and their parts
    tol_dq = scale * (err_ds + n * E24 * mag) @ kk.abs() + u * res[2].abs()
    tk = scale * (err_ds + nk * E24 * mag).transpose(2, 3) @ qq.abs()
    tv = ((factor + up + nk * E24) * p).transpose(2, 3) @ gg.abs()
    fold = lambda t: t.view(B, H // G, G, *t.shape[2:]).sum(2)
    return res, (tol_o, tol_lse, tol_dq, fold(tk) + u * res[3].abs(), fold(tv) + u * res[4].abs())


def close(got, ref, tol, what):
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(ref)), what
    err = torch.where(torch.isinf(ref), 0.0, (got - ref).abs())
    assert not torch.isnan(err).any(), what
    bad = err > tol * 1.001 + 1e-30
    assert not bool(bad.any()), (what, float((err / (tol + 1e-30)).max()))


# B, H, Hkv, L, D, window, sinks, dtype, strided, first keys
TRAIN = [
    (1, 2, 1, 1, 64, 1, 0, BF16, False, None),
    (1, 4, 2, 130, 128, 17, 4, BF16, False, None),
    (2, 4, 1, 300, 64, 64, 1, F16, True, None),
    (1, 2, 2, 257, 128, 1000, 3, BF16, True, None),      # causal attention
    (1, 3, 1, 200, 64, 1, 0, BF16, False, None),         # itself alone
    (1, 2, 1, 515, 64, 100, 130, F16, False, None),      # sinks over two key blocks
    (3, 2, 1, 190, 128, 33, 5, BF16, True, [0, 77, 190]),  # left padding, one row of nothing
    (2, 2, 2, 150, 64, 40, 3, F16, False, [149, 1]),
    (1, 4, 2, 300, 96, 60, 4, BF16, True, None),
    (1, 2, 1, 140, 80, 50, 2, F16, False, None),
    (1, 2, 1, 70, 8, 20, 2, BF16, False, None),
    (2, 2, 1, 200, 64, 50, 4, F32, True, [3, 120]),
    (1, 2, 2, 260, 128, 100, 1, F32, False, None),
    (1, 1, 1, 90, 20, 30, 0, F32, False, None),
    (1, 8, 1, 1200, 64, 90, 2, BF16, False, None),       # sinks' rows cut in many parts
]


def make(B, H, Hkv, Lq, Lk, D, dtype, strided, seed):
    gen = torch.Generator().manual_seed(seed)
    q = rows(B, H, Lq, D, dtype, gen, strided)
    k = rows(B, Hkv, Lk, D, dtype, gen, strided)
    v = rows(B, Hkv, Lk, D, dtype, gen, strided)
    return q, k, v, gen


@pytest.mark.parametrize("B,H,Hkv,L,D,W,S,dtype,strided,first", TRAIN)
def test_whole_sequences(B, H, Hkv, L, D, W, S, dtype, strided, first):
    q, k, v, gen = make(B, H, Hkv, L, L, D, dtype, strided, 0)
    g = rows(B, H, L, D, dtype, gen, True)
    f = torch.zeros(B, dtype=torch.int64) if first is None else torch.tensor(first)
    seen = window_mask(torch.arange(L).expand(B, L), f, L, W, S)
    scale = D ** -0.5
    ref, tol = bounds(q, k, v, seen, scale, dtype, g)
    qd, kd, vd, gd = (to_dev(t) for t in (q, k, v, g))
    fd = None if first is None else f.to(DEV)
    o, lse = sink_window_attention_fwd(qd, kd, vd, W, S, scale, first_key=fd)
    assert o.shape == (B, L, H, D) and o.dtype == dtype
    close(o.transpose(1, 2), ref[0], tol[0], "o")
    close(lse, ref[1], tol[1], "lse")
    again, none = sink_window_attention_fwd(qd, kd, vd, W, S, scale, first_key=fd,
                                            return_lse=False)
    assert none is None and torch.equal(again, o)
    grads = sink_window_attention_bwd(qd, kd, vd, o, lse, gd.transpose(1, 2), W, S, scale,
                                      first_key=fd)
    for got, r, t, what in zip(grads, ref[2:], tol[2:], ("dq", "dk", "dv")):
        assert got.dtype == dtype
        close(got, r, t, what)
    repeat = sink_window_attention_bwd(qd, kd, vd, o, lse, gd.transpose(1, 2), W, S, scale,
                                       first_key=fd)
    assert all(torch.equal(a, b) for a, b in zip(grads, repeat))


# B, H, Hkv, Lq, Lk, D, window, sinks, dtype, start of each sequence's rows, first keys
CACHE = [
    (1, 4, 1, 1, 1, 64, 10, 4, BF16, [0], None),
    (1, 32, 8, 1, 2000, 128, 300, 4, BF16, [1999], None),
    (5, 8, 2, 1, 900, 64, 100, 3, F16, [0, 899, 50, 450, 103], None),
    (2, 8, 1, 1, 700, 128, 5000, 0, BF16, [699, 340], None),
    (3, 4, 4, 1, 700, 80, 64, 200, BF16, [699, 150, 250], [0, 160, 30]),
    (1, 16, 1, 1, 5000, 64, 4000, 1, F16, [4999], None),
    (2, 6, 3, 5, 400, 128, 60, 2, BF16, [395, 0], None),    # several rows a step
    (1, 40, 2, 3, 400, 96, 60, 70, F16, [200], None),
    (2, 4, 2, 1, 600, 128, 90, 4, F32, [599, 3], None),
    (1, 8, 1, 7, 300, 20, 90, 4, F32, [290], [100]),
    (1, 4, 2, 150, 1000, 128, 200, 4, BF16, [850], None),   # chunks
    (2, 2, 1, 333, 900, 64, 90, 4, F16, [0, 500], [0, 510]),
    (1, 2, 1, 200, 500, 64, 90, 4, F32, [111], None),
]


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,W,S,dtype,start,first", CACHE)
def test_rows_of_a_cache(B, H, Hkv, Lq, Lk, D, W, S, dtype, start, first):
    q, k, v, gen = make(B, H, Hkv, Lq, Lk, D, dtype, False, 1)
    g = rows(B, H, Lq, D, dtype, gen, True)
    f = torch.zeros(B, dtype=torch.int64) if first is None else torch.tensor(first)
    pos = torch.tensor(start)[:, None] + torch.arange(Lq)
    seen = window_mask(pos, f, Lk, W, S)
    scale = D ** -0.5
    ref, tol = bounds(q, k, v, seen, scale, dtype, g)
    qd, kd, vd, gd = (to_dev(t) for t in (q, k, v, g))
    fd = None if first is None else f.to(DEV)
    o, lse = sink_window_attention_fwd(qd, kd, vd, W, S, scale, pos.to(DEV), fd)
    close(o.transpose(1, 2), ref[0], tol[0], "o")
    close(lse, ref[1], tol[1], "lse")
    for p in (pos, (pos - Lk).to(DEV)):  # on the host; counted from the cache's end
        same, _ = sink_window_attention_fwd(qd, kd, vd, W, S, scale, p, fd)
        assert torch.equal(same, o)
    if B == 1:
        same, _ = sink_window_attention_fwd(qd, kd, vd, W, S, scale, pos[0].to(DEV), fd)
        assert torch.equal(same, o)
    grads = sink_window_attention_bwd(qd, kd, vd, o, lse, gd.transpose(1, 2), W, S, scale,
                                      pos.to(DEV), fd)
    for got, r, t, what in zip(grads, ref[2:], tol[2:], ("dq", "dk", "dv")):
        close(got, r, t, what)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Lq,Lk", [(0, 260), (1, 700), (1, 20), (4, 300)])
def test_residual_of_o(dtype, Lq, Lk):
    """o plus its residual is the output in nearly twice the bits: off by the
    float32 sums' and the probabilities' error alone, which is common to both."""
    B, H, Hkv, D, W, S = 2, 4, 2, 64, 100, 3
    n = Lq or Lk
    q, k, v, gen = make(B, H, Hkv, n, Lk, D, dtype, False, 7)
    pos = None if not Lq else torch.tensor([Lk - n, 9])[:, None] + torch.arange(n)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    o, lse, res = sink_window_attention_fwd(qd, kd, vd, W, S, 0.125, pos, return_residual=True)
    o2, lse2 = sink_window_attention_fwd(qd, kd, vd, W, S, 0.125, pos)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    assert res.shape == o.shape and res.dtype == dtype
    u = torch.finfo(dtype).eps / 2
    # half a step of o, and the residual's own rounding
    assert bool((res.float().abs() <= u * o.float().abs() * (1 + 2 * u) + 1e-7).all())
    assert float(res.float().abs().max()) > 0 or n * H < 3
    # the same values, without the outputs' rounding, from float32 inputs: apart
    # by the probabilities' rounding only
    seen = window_mask(torch.arange(n).expand(B, n) if pos is None else pos,
                       torch.zeros(B, dtype=torch.int64), Lk, W, S)
    ref, tol = bounds(q, k, v, seen, 0.125, dtype)
    full = (o.double() + res.double()).transpose(1, 2).cpu()
    assert bool(((full - ref[0]).abs() <= (tol[0] - u * ref[0].abs()) * 1.001
                 + u * u * ref[0].abs() * 2 + 1e-7).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Lq", [1, 5, 190])
def test_rows_without_a_place(dtype, Lq):
    """Rows past the cache, or that do not follow their sequence's first one,
    give NaN; the others are not touched by them."""
    B, H, Hkv, Lk, D, W, S = 3, 4, 2, 200, 64, 30, 2
    q, k, v, _ = make(B, H, Hkv, Lq, Lk, D, dtype, False, 2)
    start = torch.tensor([Lk - (Lq + 1) // 2, 5, -Lk - 1])
    pos = start[:, None] + torch.arange(Lq)
    ok = torch.ones(B, Lq, dtype=torch.bool)
    ok[0] = pos[0] < Lk
    ok[2] = False
    if Lq > 3:
        pos[1, 3] = 5
        ok[1, 3] = False
    seen = window_mask(torch.where(ok, pos, 0), torch.zeros(B, dtype=torch.int64), Lk, W, S)
    ref, tol = bounds(q, k, v, seen, D ** -0.5, dtype)
    o, lse = sink_window_attention_fwd(q.to(DEV), k.to(DEV), v.to(DEV), W, S, D ** -0.5,
                                       pos.to(DEV))
    o = o.transpose(1, 2).cpu()
    assert torch.equal(torch.isnan(o).all(-1), ~ok[:, None].expand(B, H, Lq))
    assert torch.equal(torch.isnan(lse.cpu()), ~ok[:, None].expand(B, H, Lq))
    m = ok[:, None, :, None]
    close(torch.where(m, o, 0.0), torch.where(m, ref[0], 0.0), tol[0], "o")


def plant(t, where, gen):
    """Inf, -Inf and NaN at some dims of the rows `where` ([B, n] bool)."""
    t = t.clone()
    vals = torch.tensor([math.inf, -math.inf, math.nan])
    for b, r in torch.nonzero(where).tolist():
        h = int(torch.randint(t.shape[1], (1,), generator=gen))
        d = int(torch.randint(t.shape[3], (1,), generator=gen))
        t[b, h, r, d] = vals[int(torch.randint(3, (1,), generator=gen))].to(t.dtype)
    return t


@pytest.mark.parametrize("dtype,Lq", [(BF16, 0), (F16, 0), (F32, 0), (BF16, 1), (F32, 1), (F16, 6)])
def test_hidden_nonfinite_values_reach_nothing(dtype, Lq):
    """Left padding and the rows behind the last position filled with Inf and
    NaN: every result is that of finite padding, bit for bit where nothing was
    computed again and within the bounds elsewhere."""
    B, H, Hkv, L, D, W, S = 2, 4, 2, 300, 64, 50, 3
    f = torch.tensor([70, 11])
    n = Lq or L
    q, k, v, gen = make(B, H, Hkv, n, L, D, dtype, False, 3)
    g = rows(B, H, n, D, dtype, gen, True)
    pos = torch.arange(L).expand(B, L) if not Lq else \
        torch.tensor([140, 260])[:, None] + torch.arange(n)
    seen = window_mask(pos, f, L, W, S)
    ref, tol = bounds(q, k, v, seen, D ** -0.5, dtype, g)
    hidden = ~seen.any(1)                       # keys that no row sees
    if not Lq:                                  # rows that see nothing hold anything too
        q = plant(q, pos < f[:, None], gen)
        g = plant(g, pos < f[:, None], gen)
    k, v = plant(k, hidden, gen), plant(v, hidden, gen)
    qd, kd, vd, gd = (to_dev(t) for t in (q, k, v, g))
    args = (W, S, D ** -0.5, pos.to(DEV) if Lq else None, f.to(DEV))
    o, lse = sink_window_attention_fwd(qd, kd, vd, *args)
    close(o.transpose(1, 2), ref[0], tol[0], "o")
    close(lse, ref[1], tol[1], "lse")
    got = sink_window_attention_bwd(qd, kd, vd, o, lse, gd.transpose(1, 2), *args)
    for x, r, t, what in zip(got, ref[2:], tol[2:], ("dq", "dk", "dv")):
        close(x, r, t, what)


@pytest.mark.parametrize("dtype,Lq", [(BF16, 0), (F16, 0), (F32, 0), (BF16, 2), (F32, 1)])
def test_visible_nonfinite_values_reach_their_rows(dtype, Lq):
    """A V row with an Inf or NaN: exactly the rows that see it, exactly its
    dims; a NaN in K: its rows whole; the gradients of those keys and rows
    alone."""
    B, H, Hkv, L, D, W, S = 1, 2, 1, 260, 64, 40, 2
    n = Lq or L
    q, k, v, gen = make(B, H, Hkv, n, L, D, dtype, False, 4)
    g = rows(B, H, n, D, dtype, gen, True)
    base = 0 if not Lq else 150
    pos = (base + torch.arange(n)).expand(B, n)
    v[0, 0, 140, 5] = math.inf
    v[0, 0, 141, 5] = math.inf
    v[0, 0, 141, 6] = -math.inf
    v[0, 0, 1, 9] = math.nan       # a sink
    k[0, 0, 30, 3] = math.nan
    seen = window_mask(pos, torch.zeros(B, dtype=torch.int64), L, W, S)
    args = (W, S, D ** -0.5, pos.to(DEV) if Lq else None)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    o, lse = sink_window_attention_fwd(qd, kd, vd, *args)
    o = o.transpose(1, 2).float().cpu()
    knan = seen[0, :, 30]
    want = torch.zeros(n, D)
    want[seen[0, :, 140] | seen[0, :, 141], 5] = math.inf
    want[seen[0, :, 141], 6] = -math.inf
    want[seen[0, :, 1], 9] = math.nan
    want[knan] = math.nan
    for h in range(H):
        assert torch.equal(torch.isnan(o[0, h]), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(torch.isinf(o[0, h]), inf) and torch.equal(o[0, h][inf], want[inf])
    if Lq:
        return
    dq, dk, dv = sink_window_attention_bwd(qd, kd, vd, torch.nan_to_num(o, 0, 0, 0).transpose(1, 2)
                                           .to(dtype).to(DEV), lse, g.to(DEV).transpose(1, 2),
                                           *args)
    bad_rows = seen[0][:, [140, 141, 1, 30]].any(-1)
    good = ~bad_rows
    assert torch.isfinite(dq[0, :, good.to(DEV)]).all() and int(good.sum()) > 0
    touched = (seen[0] & bad_rows[:, None]).any(0)     # keys that a spoilt row sees
    assert torch.isfinite(dk[0, 0, ~touched]).all() and torch.isfinite(dv[0, 0, ~touched]).all()


def test_far_rows_of_a_long_cache():
    """One kv head's rows lie past 2^31 elements: a step, a chunk and their
    gradients at the far end equal those of a copy of the last keys."""
    L, D, W = 16400, 64, 100
    stride = 1 << 17               # elements: the last row starts at 2.1e9
    base = torch.empty(L * stride, dtype=BF16, device=DEV)
    k = base.as_strided((1, 1, L, D), (L * stride, L * stride, stride, 1))
    v = base[64:].as_strided((1, 1, L, D), (L * stride, L * stride, stride, 1))
    gen = torch.Generator(device=DEV).manual_seed(5)
    for t in (k, v):
        t.copy_(torch.randn(1, 1, L, D, generator=gen, device=DEV))
    for n in (1, 200):
        q = torch.randn(1, 2, n, D, generator=gen, device=DEV).to(BF16)
        g = torch.randn(1, n, 2, D, generator=gen, device=DEV).to(BF16)
        pos = torch.arange(L - n, L, device=DEV)
        res = []
        for kk, vv in ((k, v), (k.contiguous(), v.contiguous())):
            o, lse = sink_window_attention_fwd(q, kk, vv, W, 4, 0.125, pos)
            res.append((o, lse, *sink_window_attention_bwd(q, kk, vv, o, lse, g, W, 4, 0.125, pos)))
        assert all(torch.equal(a, b) for a, b in zip(*res))


def test_module_calls():
    """The module's forms: autograd against the calls on tensors, GQA, several
    sequences at their own positions, empty calls."""
    layer = SinkWindowAttention(6, 64, 32, num_sinks=3, num_key_value_heads=2).to(DEV)
    q, k, v, gen = make(2, 6, 2, 100, 100, 64, BF16, True, 6)
    qd, kd, vd = (to_dev(t).requires_grad_() for t in (q, k, v))
    out, none = layer(qd, kd, vd)
    assert none is None and out.shape == (2, 100, 384)
    g = torch.randn(2, 100, 384, generator=gen).to(BF16).to(DEV)
    out.backward(g)
    with torch.no_grad():
        o, lse, res = sink_window_attention_fwd(qd, kd, vd, 32, 3, 0.125, return_residual=True)
        want = sink_window_attention_bwd(qd, kd, vd, o, lse, g.view(2, 100, 6, 64), 32, 3, 0.125,
                                         o_residual=res)
        assert torch.equal(out, o.view(2, 100, 384)) and torch.equal(layer(qd, kd, vd)[0], out)
    for t, w in zip((qd, kd, vd), want):
        assert torch.equal(t.grad, w)
    # an expanded gradient, as a sum's backward gives it
    qd.grad = None
    layer(qd, kd, vd)[0].sum().backward()
    ones = torch.ones(2, 100, 6, 64, dtype=BF16, device=DEV)
    assert torch.equal(qd.grad, sink_window_attention_bwd(
        qd.detach(), kd.detach(), vd.detach(), o, lse, ones, 32, 3, 0.125, o_residual=res)[0])
    with torch.no_grad():
        assert layer(qd[:, :, :0], kd, vd)[0].shape == (2, 0, 384)
        assert layer(qd[:0], kd[:0], vd[:0])[0].shape == (0, 100, 384)
        assert layer(qd[:, :, :0], kd[:, :, :0], vd[:, :, :0])[0].shape == (2, 0, 384)
        gone = layer(qd[:, :, :2], kd[:, :, :0], vd[:, :, :0],
                     cache_position=torch.zeros(2, dtype=torch.int64, device=DEV))[0]
        assert torch.isnan(gone).all()


def test_refusals():
    layer = SinkWindowAttention(4, 64, 32, num_key_value_heads=2)
    q = torch.zeros(2, 4, 8, 64, dtype=BF16, device=DEV)
    k = torch.zeros(2, 2, 8, 64, dtype=BF16, device=DEV)
    with pytest.raises(RuntimeError):
        layer(q.cpu(), k.cpu(), k.cpu())
    for bad in (lambda: layer(q, k, k.float()), lambda: layer(q[:, :2], k, k),
                lambda: layer(q, k[:, :, :4], k[:, :, :4]),
                lambda: layer(q[..., :32], k[..., :32], k[..., :32]),
                lambda: layer(q, k, k, first_key=torch.zeros(3, dtype=torch.int64)),
                lambda: layer(q, k, k, first_key=torch.zeros(2)),
                lambda: layer(q, k, k, cache_position=torch.arange(7)),
                lambda: layer(q, k, k, cache_position=torch.tensor([0, 1, 2, 3, 4, 5, 7, 6])),
                lambda: layer(q, k, k, kv_cache=(k, k)),
                lambda: SinkWindowAttention(4, 64, 0), lambda: SinkWindowAttention(4, 64, 8, -1),
                lambda: SinkWindowAttention(4, 64, 8, num_key_value_heads=3),
                lambda: SinkWindowAttention(4, 256, 8), lambda: SinkWindowAttention(4, 66, 8)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        layer(q, k, k, cache_position=torch.arange(1, 9))
    with pytest.raises(RuntimeError):  # 16-bit heads are read 8 elements at a time
        sink_window_attention_fwd(q[..., :20], k[..., :20], k[..., :20], 4, 0, 1.0)
    with pytest.raises(RuntimeError):
        sink_window_attention_fwd(q, k, k, 4, 0, -1.0)


@pytest.mark.parametrize("kind", ["window", "elastic"])
def test_a_model_layer_in_steps(kind):
    """Norm, rotation, caches and attention together: a prompt in one call, the
    same prompt in chunks, then single tokens against the caches, equal the
    whole sequence in one call."""
    B, H, Hkv, L, D, dtype = 2, 8, 2, 150, 64, BF16
    rotary = QKNormRope(D, base=1e6).to(DEV).to(dtype)
    if kind == "window":
        layer = SinkWindowAttention(H, D, 40, 4, Hkv, rotary=rotary)
    else:
        layer = ElasticSparseAttention(3, 6, H, D, 16, L, Hkv, rotary=rotary)
    layer = layer.to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn(B, L, H + 2 * Hkv, D, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    with torch.no_grad():
        whole, _ = layer(q, k, v)
        kc = torch.zeros(B, Hkv, L, D, dtype=dtype, device=DEV)
        vc = torch.zeros_like(kc)
        parts, at = [], 0
        for n in (100, 37, 1, 1, 1, 10):
            pos = torch.arange(at, at + n, device=DEV)
            rows_ = slice(at, at + n)
            parts.append(layer(q[:, :, rows_], k[:, :, rows_], v[:, :, rows_],
                               cache_position=pos, kv_cache=(kc, vc))[0])
            at += n
        steps = torch.cat(parts, 1)
        yq, yk = rotary(q, k, torch.arange(L))
        assert torch.equal(kc, yk) and torch.equal(vc, v)
    # the same products in another order: probabilities rounded to bf16 each
    # time (2 u of sum p |v| <= 2 u max |v|), one rounding of the output
    u = torch.finfo(dtype).eps / 2
    lim = (4 * u + 2 * u) * float(v.abs().max())
    assert float((steps.float() - whole.float()).abs().max()) <= lim
    if kind == "window":
        seen = window_mask(torch.arange(L).expand(B, L), torch.zeros(B, dtype=torch.int64), L,
                           40, 4)
        ref, tol = bounds(yq.cpu(), yk.cpu(), v.cpu(), seen, D ** -0.5, dtype)
        for got in (steps, whole):
            close(got.view(B, L, H, D).transpose(1, 2), ref[0], tol[0], "o")
    # and training through all of it
    qg, kg, vg = (t.detach().clone().requires_grad_() for t in (q, k, v))
    out, _ = layer(qg, kg, vg)
    out.float().square().sum().backward()
    for t in (qg, kg, vg, rotary.q_weight, rotary.k_weight):
        assert t.grad is not None and torch.isfinite(t.grad).all() and bool((t.grad != 0).any())
    with pytest.raises(ValueError):
        layer(q, k, v, cache_position=torch.arange(L))
    with pytest.raises(ValueError):
        layer(q, k, v, kv_cache=(kc, vc))


def test_replayed_graph_and_another_stream():
    """A step of a layer (append, attention), a prefill and a backward captured
    and replayed on new inputs, with eager calls between; two graphs side by
    side; then another stream."""
    B, H, Hkv, L, D = 2, 8, 2, 3000, 64
    rotary = QKNormRope(D).to(DEV).to(BF16)
    layer = SinkWindowAttention(H, D, 1500, 4, Hkv, rotary=rotary).to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(9)

    def new(*s):
        return torch.randn(*s, generator=gen, device=DEV).to(BF16)

    q1, k1, v1 = new(B, H, 1, D), new(B, Hkv, 1, D), new(B, Hkv, 1, D)
    kc, vc = new(B, Hkv, L, D), new(B, Hkv, L, D)
    pos = torch.tensor([[2999], [1000]], device=DEV)
    q, g = new(B, H, 300, D), new(B, 300, H, D)

    def step():
        with torch.no_grad():
            return (layer(q1, k1, v1, cache_position=pos, kv_cache=(kc, vc))[0],)

    def train():
        o, lse = sink_window_attention_fwd(q, kc, vc, 50, 2, 0.125)
        return (o, lse, *sink_window_attention_bwd(q, kc, vc, o, lse, g, 50, 2, 0.125))

    step(), train()
    torch.cuda.synchronize()
    graphs = []
    for work in (step, train):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        graphs.append((graph, work, out))
    for _ in range(3):
        for t in (q1, k1, v1, q, g):
            t.copy_(new(*t.shape))
        for graph, work, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for _, _, out in graphs]
        for (_, work, _), have in zip(graphs, got):
            assert all(torch.equal(a, b) for a, b in zip(have, work()))
    want = train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        have = train()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(have, want))


def random_case(seed):
    """One call over everything that a call may vary."""
    import random
    r = random.Random(seed)
    B, Hkv, G = r.choice([1, 2, 3]), r.choice([1, 2]), r.choice([1, 2, 3, 5])
    dtype = r.choice([BF16, BF16, F16, F32])
    D = r.choice([8, 24, 64, 72, 104, 128]) if dtype != F32 else r.choice([4, 20, 64, 100, 128])
    Lk = r.choice([1, 31, 127, 129, 400, 641, 1100])
    Lq = Lk if r.random() < 0.5 else r.choice([1, 2, 9, 33, 128, Lk])
    Lq = min(Lq, Lk)
    start = [0] * B if Lq == Lk else [r.randint(0, Lk - Lq) for _ in range(B)]
    first = None if r.random() < 0.5 else [r.choice([0, r.randint(0, Lk), Lk]) for _ in range(B)]
    W = r.choice([1, 5, 32, 33, 100, 128, 500, 1 << 20])
    S = r.choice([0, 1, 4, 31, 128, 200])
    return B, Hkv * G, Hkv, Lq, Lk, D, W, S, dtype, start, first, r.random() < 0.5


def gradual(q, k, v, g, seen, scale, dtype):
    """What the bounds take on where values fall below the type's normal range
    (float16: 2^-14).  Spacing there is smallest_normal * eps whatever the value,
    so a rounding is off by up to half of that, `least` (2^-25), not u |x|: each
    output by least, and a product of probabilities or dS by least times the sum
    of what they meet (the forward's probabilities are divided by a sum >= 1)."""
    t = torch.finfo(dtype)
    least = t.smallest_normal * t.eps / 2
    G = q.shape[1] // k.shape[1]
    B, H, Lq, D = q.shape
    kk, vv = (x.double().abs().repeat_interleave(G, 1) for x in (k, v))
    vis = seen[:, None].double()
    fold = lambda x: x.view(B, H // G, G, *x.shape[2:]).sum(2)
    o, dq = least * (1 + vis @ vv), least * (1 + scale * (vis @ kk))
    dk = least * (1 + fold(scale * (vis.transpose(2, 3) @ q.double().abs())))
    dv = least * (1 + fold(vis.transpose(2, 3) @ g.double().abs()))
    return o, 0.0, dq, dk, dv


def run_case(B, H, Hkv, Lq, Lk, D, W, S, dtype, start, first, strided, seed):
    q, k, v, gen = make(B, H, Hkv, Lq, Lk, D, dtype, strided, seed)
    g = rows(B, H, Lq, D, dtype, gen, True)
    f = torch.zeros(B, dtype=torch.int64) if first is None else torch.tensor(first)
    pos = torch.tensor(start)[:, None] + torch.arange(Lq)
    seen = window_mask(pos, f, Lk, W, S)
    ref, tol = bounds(q, k, v, seen, D ** -0.5, dtype, g)
    tol = [a + b for a, b in zip(tol, gradual(q, k, v, g, seen, D ** -0.5, dtype))]
    qd, kd, vd, gd = (to_dev(t) for t in (q, k, v, g))
    fd = None if first is None else f.to(DEV)
    p = None if Lq == Lk else pos.to(DEV)
    o, lse, res = sink_window_attention_fwd(qd, kd, vd, W, S, D ** -0.5, p, fd,
                                            return_residual=True)
    close(o.transpose(1, 2), ref[0], tol[0], "o")
    close(lse, ref[1], tol[1], "lse")
    grads = sink_window_attention_bwd(qd, kd, vd, o, lse, gd.transpose(1, 2), W, S, D ** -0.5, p,
                                      fd, res)
    for got, r, t, what in zip(grads, ref[2:], tol[2:], ("dq", "dk", "dv")):
        close(got, r, t, what)


@pytest.mark.parametrize("seed", range(24))
def test_random_calls(seed):
    case = random_case(seed)
    print(case, flush=True)
    run_case(*case, seed)


def test_gradients_of_gradients_and_other_devices_are_refused():
    layer = SinkWindowAttention(2, 64, 8)
    q = torch.randn(1, 2, 5, 64, dtype=BF16, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(layer(q, q, q)[0].float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().square().sum().backward()
    q = q.detach()
    o, lse = sink_window_attention_fwd(q, q, q, 8, 0, 0.125)
    for bad in ((o.cpu(), lse, o), (o, lse.cpu(), o), (o, lse, o.cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            sink_window_attention_bwd(q, q, q, *bad, 8, 0, 0.125)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_broadcast_inputs(dtype, D):
    """One key and value row set for every sequence and head, one query row set
    for every sequence: the calls see views of stride 0, as their copies."""
    B, H, Hkv, L = 3, 4, 2, 150
    gen = torch.Generator().manual_seed(21)
    q1 = torch.randn(1, H, L, D, generator=gen).to(dtype).to(DEV).requires_grad_()
    k1 = torch.randn(1, 1, L, D, generator=gen).to(dtype).to(DEV).requires_grad_()
    v1 = torch.randn(B, Hkv, 1, D, generator=gen).to(dtype).to(DEV).requires_grad_()
    g = torch.randn(B, L, H * D, generator=gen).to(dtype).to(DEV)
    layer = SinkWindowAttention(H, D, 40, 3, Hkv)

    def grads(copy):
        q, k, v = (t.expand(B, h, L, D) for t, h in ((q1, H), (k1, Hkv), (v1, Hkv)))
        if copy:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        o = layer(q, k, v)[0]
        return (o.detach(), *torch.autograd.grad(o, (q1, k1, v1), g))

    for a, b in zip(grads(False), grads(True)):
        assert a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk", [(4100, 8, 1, 1, 3), (1, 600, 3, 1, 40), (1, 70, 70, 2, 2),
                                           (2000, 2, 2, 3, 3)])
def test_many_sequences_and_heads(B, H, Hkv, Lq, Lk):
    D, W, S = 64, 3, 1
    gen = torch.Generator().manual_seed(22)
    q, k, v = (torch.randn(B, h, n, D, generator=gen).to(BF16)
               for h, n in ((H, Lq), (Hkv, Lk), (Hkv, Lk)))
    pos = (Lk - Lq + torch.arange(Lq)).expand(B, Lq)
    seen = window_mask(pos, torch.zeros(B, dtype=torch.int64), Lk, W, S)
    ref, tol = bounds(q, k, v, seen, D ** -0.5, BF16)
    rotary = QKNormRope(D).to(DEV).to(BF16)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    o, lse = sink_window_attention_fwd(qd, kd, vd, W, S, D ** -0.5, pos.to(DEV))
    close(o.transpose(1, 2), ref[0], tol[0], "o")
    close(lse, ref[1], tol[1], "lse")
    # the whole step, against the rotation and the attention by themselves
    layer = SinkWindowAttention(H, D, W, S, Hkv, rotary=rotary)
    caches = torch.zeros_like(kd), torch.zeros_like(vd)
    with torch.no_grad():
        got = layer(qd, kd[:, :, -Lq:], vd[:, :, -Lq:], cache_position=pos.to(DEV),
                    kv_cache=caches)[0]
        yq, yk = rotary(qd, kd[:, :, -Lq:], pos.to(DEV))
    want_k, want_v = torch.zeros_like(kd), torch.zeros_like(vd)
    want_k[:, :, -Lq:], want_v[:, :, -Lq:] = yk, vd[:, :, -Lq:]
    assert torch.equal(caches[0], want_k) and torch.equal(caches[1], want_v)
    want, _ = sink_window_attention_fwd(yq, want_k, want_v, W, S, D ** -0.5, pos.to(DEV))
    assert torch.equal(got, want.view(B, Lq, H * D))


def test_two_threads_on_two_streams():
    """Steps, prefills and backward passes of two threads at once, each on its
    own stream, are what each gives alone."""
    import threading
    D, H, Hkv = 64, 4, 2
    rotary = QKNormRope(D).to(DEV).to(BF16)
    layer = SinkWindowAttention(H, D, 90, 4, Hkv, rotary=rotary)

    def work(seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        new = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(BF16)
        kc, vc = new(2, Hkv, 700, D), new(2, Hkv, 700, D)
        out = []
        for i in range(6):
            n = (1, 5, 140)[i % 3]
            q, k, v = new(2, H, n, D), new(2, Hkv, n, D), new(2, Hkv, n, D)
            with torch.no_grad():
                at = torch.arange(n, device=DEV) + 100 * i
                out.append(layer(q, k, v, cache_position=at, kv_cache=(kc, vc))[0])
            q, k, v = (t.requires_grad_() for t in (q, k, v))
            o = layer(q, k, v)[0]
            out += [o.detach(), *torch.autograd.grad(o, (q, k, v), torch.ones_like(o))]
        return out

    want = [work(s) for s in (1, 2)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = work(i + 1)
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert a is not None and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("H,L,D,W,S,dtype", [
    (16, 1500, 128, 200, 4, BF16), (12, 1111, 64, 300, 130, F16), (24, 700, 64, 700, 0, BF16),
    (8, 900, 64, 120, 4, F32)])
def test_many_heads_on_one_kv_head(H, L, D, W, S, dtype):
    """Few key blocks with many rows each: all of them cut into chunks."""
    run_case(1, H, 1, L, L, D, W, S, dtype, [0], None, True, 31)


@pytest.mark.parametrize("dtype,D,Lq,W", [(BF16, 128, 300, 5000), (F16, 64, 513, 3000),
                                          (BF16, 72, 300, 5000), (F32, 64, 600, 5000)])
def test_blocks_cut_into_key_ranges(dtype, D, Lq, W):
    """A chunk of few heads over a long cache: row blocks whose keys are walked
    in ranges side by side, with left padding, Inf and NaN where no row looks, one
    visible Inf, rows without a place, and from a graph."""
    H, Lk, S, first = 4, 5000, 3, 700
    q, k, v, gen = make(1, H, 1, Lq, Lk, D, dtype, False, 41)
    pos = Lk - 90 - Lq + torch.arange(Lq)[None]
    f = torch.tensor([first])
    seen = window_mask(pos, f, Lk, W, S)
    scale = D ** -0.5
    ref, tol = bounds(q, k, v, seen, scale, dtype)
    hidden = ~seen.any(1)
    k, v = plant(k, hidden, gen), plant(v, hidden, gen)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    args = (W, S, scale, pos.to(DEV), f.to(DEV))
    o, lse, res = sink_window_attention_fwd(qd, kd, vd, *args, return_residual=True)
    close(o.transpose(1, 2), ref[0], tol[0], "o")
    close(lse, ref[1], tol[1], "lse")
    if res is not None:
        u = torch.finfo(dtype).eps / 2
        both = (o.double() + res.double()).transpose(1, 2).cpu()
        assert bool(((both - ref[0]).abs() <= tol[0] + u * u * ref[0].abs() + 2.0 ** -24).all())
    assert torch.equal(sink_window_attention_fwd(qd, kd, vd, *args, return_lse=False)[0], o)
    vi = vd.clone()
    vi[0, 0, Lk - 90 - Lq, 5] = math.inf  # the first row's own key: every row's, or the window's
    oi, li = sink_window_attention_fwd(qd, kd, vi, *args)
    sees = seen[0, :, Lk - 90 - Lq].to(DEV)
    assert torch.isposinf(oi[0, sees, :, 5]).all() and torch.isfinite(oi[0, :, :, 6:]).all()
    assert torch.equal(li, lse) or torch.allclose(li, lse, rtol=1e-5, atol=1e-5)
    late = pos.to(DEV) + 120             # the last rows past the cache's end
    ol, ll = sink_window_attention_fwd(qd, torch.nan_to_num(kd), torch.nan_to_num(vd), W, S, scale,
                                       late, f.to(DEV))
    out = (late[0] >= Lk)
    assert out.any() and torch.isnan(ol[0, out]).all() and torch.isnan(ll[0, :, out]).all()
    # (keys behind pos hold anything, what nan_to_num makes of Inf among it: q k
    # overflows there, and the formula gives NaN; rows before them are finite)
    assert torch.isfinite(ol[0, late[0] <= int(pos.max())]).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        og, lg, _ = sink_window_attention_fwd(qd, kd, vd, *args, return_residual=True)
    for _ in range(3):
        og.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(og, o) and torch.equal(lg, lse)
        sink_window_attention_fwd(qd, kd, vi, *args)

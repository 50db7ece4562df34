"""Norm and rotation of queries and keys (esa_qk_norm_rope_*) against float64
(GPU).

Tolerances.  An output is rounded once: u |y|, u = finfo(dtype).eps / 2.  Before
that, float32: the sum of squares in lanes and shuffles (under 20 roundings of
2^-24, halved by the root), the gain's and the cosines' products, cosines off
by at most 4 * 2^-24 (the turn rounded to float32, then sincospif): under
40 * 2^-24 of the pair's two products together.  The gains' gradients are sums
of N terms: every lane adds its rows in turn, then 32 lanes, then up to eight
parts a lane of the second kernel and 7 steps of its tree.
"""
import pytest
import torch

from layer_oracle import norm_rope, norm_rope_bwd
from qk_norm_rope import (QKNormRope, qk_norm_rope_append, qk_norm_rope_bwd, qk_norm_rope_fwd)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E24 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rows(B, heads, n, D, dtype, gen, layout):
    if layout == "bhld":
        t = torch.randn(B, heads, n, D, generator=gen)
    else:
        t = torch.randn(B, n, heads, D, generator=gen).transpose(1, 2)
    return t.to(dtype)


def on_dev(t, layout):
    """t on the device in the same memory order (fused: a view with room
    between the rows)."""
    if layout == "fused":
        B, H, n, D = t.shape
        x = torch.full((B, n, H + 3, D), float("nan"), dtype=t.dtype, device=DEV)
        x[:, :, 1:H + 1] = t.transpose(1, 2).to(DEV)
        return x[:, :, 1:H + 1].transpose(1, 2)
    if layout == "blhd":
        return t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    return t.contiguous().to(DEV)


def pair_size(x, gain, eps, rd, interleaved):
    """|a| + |b| of each element's pair before the rotation."""
    x = x.double()
    y = (x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)).abs()
    y = y * (1.0 if gain is None else gain.double().abs())
    z = y.clone()
    if interleaved:
        s = y[..., 0:rd:2] + y[..., 1:rd:2]
        z[..., 0:rd:2] = s
        z[..., 1:rd:2] = s
    else:
        s = y[..., :rd // 2] + y[..., rd // 2:rd]
        z[..., :rd // 2] = s
        z[..., rd // 2:rd] = s
    return z


def close(got, ref, tol):
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{float((err / tol.clamp(min=1e-300)).max())} of the bound"


SHAPES = [
    # B, H, Hkv, n, D, rotary_dim, interleaved, dtype, layout
    (1, 32, 8, 1, 128, 128, False, BF16, "bhld"),
    (2, 4, 2, 37, 128, 128, False, BF16, "fused"),
    (1, 3, 1, 130, 64, 64, True, F16, "blhd"),
    (3, 2, 2, 17, 96, 64, False, F16, "fused"),
    (2, 5, 5, 9, 80, 80, False, BF16, "bhld"),
    (1, 2, 1, 33, 72, 72, False, BF16, "blhd"),    # halves of 36: 8-byte pieces
    (1, 2, 1, 33, 72, 72, True, F16, "blhd"),
    (1, 2, 1, 21, 20, 8, False, BF16, "bhld"),     # head_dim no multiple of 8
    (1, 2, 2, 40, 256, 256, False, BF16, "bhld"),
    (1, 2, 1, 40, 256, 32, True, F32, "fused"),
    (2, 3, 1, 19, 128, 128, False, F32, "blhd"),
    (1, 1, 1, 5, 8, 8, False, F32, "bhld"),
    (1, 16, 4, 3000, 64, 64, False, BF16, "fused"),
]


def case(B, H, Hkv, n, D, rd, dtype, layout, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q = rows(B, H, n, D, dtype, gen, layout) * 3
    k = rows(B, Hkv, n, D, dtype, gen, layout)
    wq = (1 + 0.2 * torch.randn(D, generator=gen)).to(dtype)
    wk = (1 + 0.2 * torch.randn(D, generator=gen)).to(dtype)
    pos = torch.randint(-50, 1 << 20, (B, n), generator=gen)
    freq = 1e4 ** (-torch.arange(rd // 2, dtype=torch.float64) / (rd // 2))
    return q, k, wq, wk, pos, freq, gen


@pytest.mark.parametrize("B,H,Hkv,n,D,rd,inter,dtype,layout", SHAPES)
def test_forward(B, H, Hkv, n, D, rd, inter, dtype, layout):
    q, k, wq, wk, pos, freq, _ = case(B, H, Hkv, n, D, rd, dtype, layout)
    yq, yk = qk_norm_rope_fwd(on_dev(q, layout), on_dev(k, layout), wq.to(DEV), wk.to(DEV),
                              freq.to(DEV), pos.to(DEV), 1e-6, inter)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.dtype == dtype
    for y, x, w in ((yq, q, wq), (yk, k, wk)):
        ref = norm_rope(x, w, pos, freq, 1e-6, inter)
        tol = unit(dtype) * ref.abs() + 40 * E24 * pair_size(x, w, 1e-6, rd, inter)
        close(y, ref, tol * 1.001 + 1e-30)


@pytest.mark.parametrize("B,H,Hkv,n,D,rd,inter,dtype,layout", SHAPES)
def test_backward(B, H, Hkv, n, D, rd, inter, dtype, layout):
    q, k, wq, wk, pos, freq, gen = case(B, H, Hkv, n, D, rd, dtype, layout, 1)
    gq = rows(B, H, n, D, dtype, gen, layout)
    gk = rows(B, Hkv, n, D, dtype, gen, "bhld")
    dq, dk, dwq, dwk = qk_norm_rope_bwd(
        on_dev(q, layout), on_dev(k, layout), wq.to(DEV), wk.to(DEV), freq.to(DEV), pos.to(DEV),
        on_dev(gq, layout), on_dev(gk, "bhld"), 1e-6, inter)
    for dx, dw, x, w, g in ((dq, dwq, q, wq, gq), (dk, dwk, k, wk, gk)):
        ref, refw, sizew = norm_rope_bwd(x, w, pos, freq, 1e-6, inter, g)
        xd = x.double()
        r = 1 / torch.sqrt(xd.square().mean(-1, keepdim=True) + 1e-6)
        gw = pair_size(g, w, 0.0, rd, inter) * torch.sqrt(g.double().square().mean(-1, keepdim=True))
        # the gradient and the mean's product, each off by under 60 roundings
        # (the mean: 20 in its sum, 40 in its terms, and the root's twice)
        size = r * (gw + (xd * r).abs() * (gw * (xd * r).abs()).mean(-1, keepdim=True))
        close(dx, ref, unit(dtype) * ref.abs() * 1.001 + 100 * E24 * size + 1e-30)
        # each term off by 60 roundings, and the sum's own
        N = x.shape[0] * x.shape[1] * x.shape[2]
        close(dw, refw, unit(dtype) * refw.abs() * 1.001 + (60 + N + 47) * E24 * sizew + 1e-30)


def test_gradients_against_differences():
    """The float32 gradients against central differences of the float64
    formula."""
    gen = torch.Generator().manual_seed(5)
    B, H, n, D, rd = 1, 2, 3, 16, 16
    q = torch.randn(B, H, n, D, generator=gen)
    k = torch.randn(B, 1, n, D, generator=gen)
    w = 1 + 0.1 * torch.randn(D, generator=gen)
    pos = torch.tensor([[3, 77, 1000]])
    freq = 1e4 ** (-torch.arange(8, dtype=torch.float64) / 8)
    gq, gk = torch.randn(B, H, n, D, generator=gen), torch.randn(B, 1, n, D, generator=gen)
    got = qk_norm_rope_bwd(q.to(DEV), k.to(DEV), w.to(DEV), w.to(DEV), freq.to(DEV), pos.to(DEV),
                           gq.to(DEV), gk.to(DEV))

    def loss(x, gain, g):
        return (norm_rope(x, gain, pos, freq, 1e-6, False) * g.double()).sum()

    step = 2.0 ** -20   # third derivatives are of order 1: the quotient is off by under 1e-9
    for x, g, dx, dw in ((q, gq, got[0], got[2]), (k, gk, got[1], got[3])):
        x, wd = x.double(), w.double()
        num = torch.zeros_like(x)
        for i in range(x.numel()):
            e = torch.zeros(x.numel(), dtype=torch.float64)
            e[i] = step
            e = e.view(x.shape)
            num.view(-1)[i] = (loss(x + e, wd, g) - loss(x - e, wd, g)) / (2 * step)
        # (float32 gradients of order 1 from under 100 roundings)
        assert float((dx.double().cpu() - num).abs().max()) < 200 * E24 * 10
        for i in range(D):
            e = torch.zeros(D, dtype=torch.float64)
            e[i] = step
            d = (loss(x, wd + e, g) - loss(x, wd - e, g)) / (2 * step)
            assert abs(float(dw[i]) - float(d)) < 200 * E24 * 10


def test_far_positions_keep_their_angles():
    """Unit rows at positions up to 2^40: the rotation against float64."""
    D = 64
    pos = torch.tensor([[0, 1, 2 ** 24 + 1, 2 ** 31 + 5, 2 ** 40 + 3, -7]])
    x = torch.ones(1, 1, 6, D)
    freq = 1e6 ** (-torch.arange(32, dtype=torch.float64) / 32)
    y, _ = qk_norm_rope_fwd(x.to(DEV), x.to(DEV), None, None, freq.to(DEV), pos.to(DEV), 0.0)
    ref = norm_rope(x, None, pos, freq, 0.0, False)
    # the angle in float64: 2^40 * 2^-53, a few roundings of it, over 2 pi
    close(y, ref, torch.full_like(ref, 2 * (40 * E24 + 8 * 2.0 ** -13)))
    near = slice(0, 3)
    close(y[:, :, near], ref[:, :, near], torch.full_like(ref[:, :, near], 2 * 41 * E24))


def test_special_rows():
    """A zero row stays 0; a NaN or Inf row stays its own."""
    D = 128
    x = torch.randn(1, 2, 8, D, generator=torch.Generator().manual_seed(2)).to(BF16)
    x[0, 0, 1] = 0
    x[0, 0, 2, 5] = float("nan")
    x[0, 1, 3, 7] = float("inf")
    freq = 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    pos = torch.arange(8)
    y, _ = qk_norm_rope_fwd(x.to(DEV), x.to(DEV), None, None, freq.to(DEV), pos.to(DEV))
    y = y.cpu()
    assert bool((y[0, 0, 1] == 0).all())
    bad = torch.zeros(1, 2, 8, dtype=torch.bool)
    bad[0, 0, 2] = bad[0, 1, 3] = True
    assert torch.equal(~torch.isfinite(y).all(-1), bad)


@pytest.mark.parametrize("inter", [False, True])
def test_elements_past_the_rotation_are_their_own(inter):
    # an infinite gain or gradient reaches its own element (and its pair's),
    # no neighbour's
    D, rd = 64, 32
    q, k, wq, wk, pos, freq, gen = case(1, 2, 1, 3, D, rd, F32, "bhld")
    wq[40] = float("inf")
    yq, _ = qk_norm_rope_fwd(q.to(DEV), k.to(DEV), wq.to(DEV), wk.to(DEV), freq.to(DEV),
                             pos.to(DEV), 1e-6, inter)
    finite = torch.isfinite(yq.cpu())
    assert not finite[..., 40].any() and int((~finite).sum()) == yq[..., 40].numel()
    gq, gk = torch.randn(q.shape, generator=gen), torch.randn(k.shape, generator=gen)
    gq[0, 0, 1, 50] = float("inf")
    _, _, dwq, _ = qk_norm_rope_bwd(q.to(DEV), k.to(DEV), wk.to(DEV), wk.to(DEV), freq.to(DEV),
                                    pos.to(DEV), gq.to(DEV), gk.to(DEV), 1e-6, inter)
    finite = torch.isfinite(dwq.cpu())
    assert not finite[50] and int((~finite).sum()) == 1


@pytest.mark.parametrize("dtype,D,rd,inter", [(BF16, 128, 128, False), (F16, 64, 32, True),
                                              (F32, 80, 80, False), (BF16, 72, 72, False)])
@pytest.mark.parametrize("n", [1, 5, 150])
def test_append(dtype, D, rd, inter, n):
    """The append writes exactly what forward gives at the rows' places, the
    values bit for bit, and nothing else of the caches."""
    B, H, Hkv, L = 3, 6, 2, 400
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(B, n, H + 2 * Hkv, D, generator=gen).to(dtype).to(DEV).transpose(1, 2)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    w = (1 + 0.1 * torch.randn(D, generator=gen)).to(dtype).to(DEV)
    freq = (1e4 ** (-torch.arange(rd // 2, dtype=torch.float64) / (rd // 2))).to(DEV)
    pos = torch.tensor([0, L - n, 123])[:, None] + torch.arange(n)
    kc = torch.randn(B, Hkv, L, D, generator=gen).to(dtype).to(DEV)
    vc = torch.randn(B, Hkv, L, D, generator=gen).to(dtype).to(DEV)
    kr, vr = kc.clone(), vc.clone()
    yq, yk = qk_norm_rope_fwd(q, k, w, w, freq, pos, 1e-6, inter)
    for b in range(B):
        kr[b, :, pos[b, 0]:pos[b, 0] + n] = yk[b]
        vr[b, :, pos[b, 0]:pos[b, 0] + n] = v[b]
    got = qk_norm_rope_append(q, k, v, kc, vc, w, w, freq, pos.to(DEV), 1e-6, inter)
    assert torch.equal(got, yq) and torch.equal(kc, kr) and torch.equal(vc, vr)
    # the same places counted from the cache's end
    kc.zero_()
    got = qk_norm_rope_append(q, k, v, kc, vc, w, w, freq, (pos - L).to(DEV), 1e-6, inter)
    assert torch.equal(got, yq)
    for b in range(B):
        assert torch.equal(kc[b, :, pos[b, 0]:pos[b, 0] + n], yk[b])


def test_append_leaves_out_rows_without_a_place():
    B, H, Hkv, n, D, L = 4, 2, 1, 3, 64, 32
    gen = torch.Generator().manual_seed(4)
    q = torch.randn(B, H, n, D, generator=gen).to(BF16).to(DEV)
    k = torch.randn(B, Hkv, n, D, generator=gen).to(BF16).to(DEV)
    kc = torch.zeros(B, Hkv, L, D, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    freq = (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    pos = torch.tensor([[30, 31, 32],       # past the end
                        [5, 5, 7],          # repeated
                        [-40, -39, -38],    # before the start
                        [1, 2, 3]])
    y = qk_norm_rope_append(q, k, k, kc, vc, None, None, freq, pos.to(DEV))
    ok = torch.tensor([[1, 1, 0], [1, 0, 1], [0, 0, 0], [1, 1, 1]], dtype=torch.bool)
    assert torch.equal(torch.isfinite(y).all(-1).all(1).cpu(), ok)
    written = torch.zeros(B, L, dtype=torch.bool)
    for b in range(B):
        for s in range(n):
            if ok[b, s]:
                written[b, pos[b, s]] = True
    assert torch.equal((vc != 0).any(-1).any(1).cpu(), written)
    assert torch.equal((kc != 0).any(-1).any(1).cpu(), written)


def test_refusals():
    layer = QKNormRope(64).to(DEV)
    q = torch.zeros(1, 4, 6, 64, dtype=BF16, device=DEV)
    k = torch.zeros(1, 2, 6, 64, dtype=BF16, device=DEV)
    c = torch.zeros(1, 2, 32, 64, dtype=BF16, device=DEV)
    pos = torch.arange(6)
    with pytest.raises(RuntimeError):
        layer(q.cpu(), k.cpu(), pos)
    with pytest.raises(ValueError):
        layer(q, k.float(), pos)
    with pytest.raises(ValueError):
        layer(q, k, torch.arange(5))
    with pytest.raises(ValueError):
        layer(q, k, pos.float())
    with pytest.raises(ValueError):
        layer(q[..., :32], k[..., :32], pos)
    with pytest.raises(ValueError):
        layer(q.double(), k.double(), pos)
    with pytest.raises(ValueError):
        layer(q, k[:, :, :5], pos)
    with pytest.raises(IndexError):
        layer.append(q, k, k, c, c.clone(), torch.arange(30, 36))
    with pytest.raises(ValueError):
        layer.append(q, k, k, c, c.clone(), torch.tensor([0, 1, 2, 3, 4, 4]))
    with pytest.raises(ValueError):
        layer.append(q, k, k[:, :1], c, c.clone(), pos)
    with pytest.raises(ValueError):
        layer.append(q, k, k, c, c[:, :, :16], pos)
    with pytest.raises(ValueError):
        layer.append(q, k, k, c[:, :1].expand(1, 2, 32, 64), c.clone(), pos)
    with pytest.raises(ValueError):
        layer.append(q.clone().requires_grad_(), k, k, c, c.clone(), pos)
    with pytest.raises(ValueError):
        QKNormRope(64, rotary_dim=12)
    with pytest.raises(ValueError):
        QKNormRope(260)


def test_module_autograd_and_empty_calls():
    layer = QKNormRope(64, rotary_dim=32, base=5e5).to(DEV)
    half = QKNormRope(64, rotary_dim=32, base=5e5).to(DEV).to(BF16)
    assert half.inv_freq.dtype == torch.float64 and half.q_weight.dtype == BF16
    g = torch.Generator(device=DEV).manual_seed(6)
    q = torch.randn(2, 4, 10, 64, generator=g, device=DEV).requires_grad_()
    k = torch.randn(2, 2, 10, 64, generator=g, device=DEV).requires_grad_()
    yq, yk = layer(q, k, torch.arange(10))
    (yq.square().sum() + (3 * yk).sum()).backward()
    want = qk_norm_rope_bwd(q.detach(), k.detach(), layer.q_weight, layer.k_weight,
                            layer.inv_freq, torch.arange(10), 2 * yq.detach(),
                            torch.full_like(yk, 3.0))
    for got, ref in zip((q.grad, k.grad, layer.q_weight.grad, layer.k_weight.grad), want):
        assert torch.equal(got, ref)
    empty = layer(q[:, :, :0].detach(), k[:, :, :0].detach(), torch.arange(0))
    assert empty[0].shape == (2, 4, 0, 64)
    q0 = torch.zeros(0, 4, 3, 64, device=DEV, requires_grad=True)
    y0, z0 = layer(q0, torch.zeros(0, 2, 3, 64, device=DEV), torch.arange(3))
    layer.q_weight.grad = None
    (y0.sum() + z0.sum()).backward()
    assert bool((layer.q_weight.grad == 0).all())


def test_replayed_graph_and_another_stream():
    """Forward, backward and append captured once and replayed on new inputs,
    eager work between; then the forward on another stream."""
    layer = QKNormRope(128).to(DEV).to(BF16)
    gen = torch.Generator(device=DEV).manual_seed(7)

    def new(*s):
        return torch.randn(*s, generator=gen, device=DEV).to(BF16)

    q, k, gq, gk = new(2, 8, 33, 128), new(2, 2, 33, 128), new(2, 8, 33, 128), new(2, 2, 33, 128)
    kc, vc = new(2, 2, 64, 128), new(2, 2, 64, 128)
    pos = torch.arange(33, device=DEV)

    def work():
        with torch.no_grad():
            y = layer(q, k, pos)
            d = qk_norm_rope_bwd(q, k, layer.q_weight, layer.k_weight, layer.inv_freq, pos, gq, gk)
            a = layer.append(q, k, k, kc, vc, pos + 7)
        return (*y, *d, a)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for _ in range(3):
        for t in (q, k, gq, gk):
            t.copy_(new(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out] + [kc.clone(), vc.clone()]
        want = list(work()) + [kc, vc]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ref = layer(q, k, pos)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer(q, k, pos)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ref)


def test_rows_in_order_without_positions():
    """No positions: row r at r, also where a layer's first call is captured
    and another length, then the captured one again, follow eagerly."""
    layer = QKNormRope(64).to(DEV).to(BF16)
    gen = torch.Generator(device=DEV).manual_seed(9)
    q = torch.randn(2, 4, 21, 64, generator=gen, device=DEV).to(BF16)
    k = torch.randn(2, 2, 21, 64, generator=gen, device=DEV).to(BF16)
    with torch.no_grad():
        want = layer(q, k, torch.arange(21))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer.attention_rows(q, k, k, None, None)
        for _ in range(3):
            got = layer.attention_rows(q, k, k, None, None)
            short = layer(q[:, :, :5], k[:, :, :5])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            assert torch.equal(short[0], want[0][:, :, :5])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_no_second_derivative():
    layer = QKNormRope(64).to(DEV)
    q = torch.randn(1, 2, 3, 64, device=DEV, requires_grad=True)
    y, _ = layer(q, q, torch.arange(3))
    (g,) = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.square().sum().backward()


@pytest.mark.parametrize("dtype,D,rd,inter,H,Hkv,n", [
    (BF16, 128, 128, False, 31, 9, 17001), (F16, 40, 32, True, 41, 3, 41000),
    (F32, 256, 64, False, 9, 4, 11003), (BF16, 72, 72, False, 1, 1, 499999)])
def test_long_rows_of_one_projection(dtype, D, rd, inter, H, Hkv, n):
    """More than the last-level cache holds, a token's heads side by side: the
    same bits as head by head, for the forward and an append."""
    gen = torch.Generator(device=DEV).manual_seed(12)
    x = torch.randn(1, n, H + 2 * Hkv, D, generator=gen, device=DEV).to(dtype)
    q, k, v = (t.transpose(1, 2) for t in x.split((H, Hkv, Hkv), 2))
    layer = QKNormRope(D, rd, base=5e5, interleaved=inter).to(DEV).to(dtype)
    pos = torch.arange(7, n + 7, device=DEV)
    with torch.no_grad():
        layer.q_weight.uniform_(0.5, 1.5)
        for a, b in zip(layer(q, k, pos), layer(q.contiguous(), k.contiguous(), pos)):
            assert torch.equal(a, b)
        caches = [[torch.zeros(1, Hkv, n + 9, D, dtype=dtype, device=DEV) for _ in "kv"]
                  for _ in range(2)]
        a = layer.append(q, k, v, *caches[0], pos)
        b = layer.append(q.contiguous(), k.contiguous(), v.contiguous(), *caches[1], pos)
    assert torch.equal(a, b)
    assert all(torch.equal(x, y) for x, y in zip(*caches))

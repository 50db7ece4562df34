"""Float64 oracles of the operators around an attention layer, on the CPU:
norm and rotation of queries and keys, and attention over a causal window with
sinks.  Written from the formulas; no code shared with the kernels."""
import math

import torch


def rotate(x, positions, inv_freq, interleaved, inverse=False):
    """x float64 [B, H, n, D], positions int64 [B, n]: the first
    2 len(inv_freq) elements' pairs turned by position * inv_freq."""
    half = inv_freq.numel()
    a = positions.double()[:, None, :, None] * inv_freq.double()
    c, s = torch.cos(a), torch.sin(a)
    if inverse:
        s = -s
    y = x.clone()
    if interleaved:
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = u * c - v * s
        y[..., 1:2 * half:2] = v * c + u * s
    else:
        u, v = x[..., :half], x[..., half:2 * half]
        y[..., :half] = u * c - v * s
        y[..., half:2 * half] = v * c + u * s
    return y


def norm_rope(x, gain, positions, inv_freq, eps, interleaved):
    """y = R(p) (x / sqrt(mean x^2 + eps) * gain), float64."""
    x = x.double()
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return rotate(n * (1.0 if gain is None else gain.double()), positions, inv_freq, interleaved)


def norm_rope_bwd(x, gain, positions, inv_freq, eps, interleaved, dy):
    """(dx, dgain, sum of |terms| of dgain) by the formulas, float64."""
    x, dy = x.double(), dy.double()
    r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r
    g = rotate(dy, positions, inv_freq, interleaved, inverse=True)
    gw = g * (1.0 if gain is None else gain.double())
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    return dx, (g * n).sum((0, 1, 2)), (g * n).abs().sum((0, 1, 2))


def window_mask(positions, first_key, kv_len, window, sinks):
    """bool [B, n, kv_len]: key j is visible to the row at position p."""
    j = torch.arange(kv_len)
    p = positions[:, :, None]
    f = first_key.clamp(0, kv_len)[:, None, None]
    return (j >= f) & (j <= p) & ((p - j < window) | (j - f < sinks))


def window_attention(q, k, v, seen, scale, dout=None):
    """Attention of q [B, H, n, D] over k, v [B, Hkv, L, D] where seen
    [B, n, L]; a row that sees nothing gives 0 (lse -inf).  Masked places are
    left out of every sum, whatever they hold.  Returns (out [B, H, n, D],
    lse) or, with dout, (out, lse, dq, dk, dv); float64."""
    B, H, n, D = q.shape
    Hkv, L = k.shape[1], k.shape[2]
    G = H // Hkv
    out = torch.zeros(B, H, n, D, dtype=torch.float64)
    lse = torch.full((B, H, n), -math.inf, dtype=torch.float64)
    dq = torch.zeros_like(out)
    dk = torch.zeros(B, Hkv, L, D, dtype=torch.float64)
    dv = torch.zeros_like(dk)
    for b in range(B):
        some = seen[b].any(0)
        cols = torch.nonzero(some)[:, 0]
        vis = seen[b][:, cols]
        empty = ~vis.any(-1)
        for h in range(H):
            kk, vv = k[b, h // G][cols].double(), v[b, h // G][cols].double()
            qq = q[b, h].double()
            s = torch.where(vis, qq @ kk.t() * scale, -math.inf)
            lse[b, h] = torch.logsumexp(s, -1)
            p = torch.where(vis, torch.softmax(s, -1), 0.0)
            p[empty] = 0.0
            o = _masked_product(p, vv, vis)
            out[b, h] = o
            if dout is None:
                continue
            g = dout[b, h].double()
            dp = torch.where(vis, g @ vv.t(), 0.0)
            ds = torch.where(vis, p * (dp - (g * o).sum(-1, keepdim=True)) * scale, 0.0)
            dq[b, h] = _masked_product(ds, kk, vis)
            dk[b, h // G].index_add_(0, cols, _masked_product(ds.t(), qq, vis.t()))
            dv[b, h // G].index_add_(0, cols, _masked_product(p.t(), g, vis.t()))
    return (out, lse) if dout is None else (out, lse, dq, dk, dv)


def _masked_product(p, x, vis):
    """p @ x with the masked terms left out (0 times a NaN there is 0)."""
    fin = torch.isfinite(x)
    if bool(fin.all()):
        return p @ x
    y = p @ torch.where(fin, x, 0.0)
    for r, d in torch.nonzero(~fin):
        rows = vis[:, r]
        y[rows, d] += p[rows, r] * x[r, d]
    return y

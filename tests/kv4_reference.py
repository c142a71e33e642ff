"""Plain 64-bit implementations of the 4-bit key/value cache's definitions, for the tests."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}


def toward_zero(x, t):
    """x >= 0 in 64 bits rounded toward zero to `t`."""
    r = x.to(t)
    return torch.where(r.double() > x, torch.nextafter(r, torch.zeros_like(r)), r).double()


def quantise(x, group):
    """x [..., D] of type T (CPU): the values that its codes stand for, and the scales [..., D / group], both in 64 bits."""
    t = x.dtype
    g = x.double().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = toward_zero((hi - lo) / 15, t)
    c = torch.where(s > 0, ((g - lo) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
    return (c * s + lo).flatten(-2).to(t).double(), s[..., 0]


def rotate(x, positions, cos_sin, interleaved):
    """x [tokens, heads, D] (CPU), in 64 bits, not rounded."""
    rot = cos_sin.shape[1]
    c, s = cos_sin.double()[positions][:, None].chunk(2, -1)
    y = x.double().clone()
    if interleaved:
        a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def attend(q, k, v, scale, causal):
    """q [n, Hq, D], k, v [m, Hk, D] in 64 bits -> (out, tolerance) for a kernel that rounds probabilities and the result
    to T once each (half a step: eps / 2), with scores and sums in 32 bits.

    The tolerance: A = sum of p |v| / sum of p is what a relative error of the probabilities is worth.
    Probabilities: eps / 2 for the rounding; 2 ds for the score errors in the probability and in the sum, where ds =
    (D + 8) 2^-23 scale sum |q k| (D products added in 32 bits with truncation) ; m 2^-23 for the sums over the keys;
    2^-20 for the exponentials.  The result: eps / 2 of itself."""
    def tolerance_for(eps):
        return (eps / 2 * (A + out.abs()) + (2 * ds + m * 2.0 ** -23 + 2.0 ** -20) * A) * (1 + 2.0 ** -6) + 2.0 ** -25

    n, hq, d = q.shape
    m, hk, _ = k.shape
    g = hq // hk
    out, A = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    ds = 0.0
    if m and n:
        kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        s = torch.einsum("nhd,mhd->hnm", q, kk) * scale
        ds = (d + 8) * 2.0 ** -23 * abs(scale) * float(torch.einsum("nhd,mhd->hnm", q.abs(), kk.abs()).max())
        if causal:
            sees = m - n + torch.arange(n)[:, None]
            s = s.masked_fill(torch.arange(m)[None] > sees, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if causal else torch.softmax(s, -1)
        out = torch.einsum("hnm,mhd->nhd", p, vv)
        A = torch.einsum("hnm,mhd->nhd", p, vv.abs())
    return out, tolerance_for

"""Plain float64 statements of the attention sublayer's operators, and the bounds of their kernels."""

from __future__ import annotations

import math

import torch


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype)


def rope(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False, dtype=torch.bfloat16):
    """(y, bound) of one of q and k [*lead, H, D]. The bound: the output's own rounding, and of its terms' sizes (those of the
    pair) what float32 leaves: the sum of D squares (16 in a row, 3 levels: 19 roundings, halved by the root), the root and
    its reciprocal (2), two products, sine and cosine (the angle's reduction 1, the series 3), two products and a sum: under
    24 of 2^-24. The angle itself is formed in float64: 2 of 2^-52 of it."""
    x = x.double().cpu()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        x = x * weight.double().cpu()
    f = inv_freq.double().cpu()
    R = 2 * f.numel()
    angle = positions.double().cpu()[..., None, None] * f
    y, size, far = x.clone(), x.abs(), torch.zeros_like(x)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = x[..., a], x[..., b]
    y[..., a] = xa * torch.cos(angle) - xb * torch.sin(angle)
    y[..., b] = xb * torch.cos(angle) + xa * torch.sin(angle)
    size[..., a] = size[..., b] = xa.abs() + xb.abs()
    far[..., a] = far[..., b] = angle.abs()
    c = 24 * 2.0**-24 + 2 * 2.0**-52 * far
    return y, half_step(dtype) * (y.abs() + c * size) + c * size


def attend(q, k, v, positions, window=None, sinks=0, scale=None):
    """One sequence in float64: q [n, Hq, D] at `positions` [n], k and v [m, Hk, D]. Returns (o, sizes of its terms
    sum_j p_j |v_j|, [n, Hq] relative error of a weight by the scores' rounding in float32)."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    n, Hq, D = q.shape
    m, Hk = k.shape[:2]
    k, v = (t.repeat_interleave(Hq // Hk, 1) for t in (k, v))
    scale = D**-0.5 if scale is None else scale
    j, p = torch.arange(m), positions.cpu().long()[:, None]
    seen = j <= p
    if window is not None:
        seen &= (p - j < window) | (j < sinks)
    o, size = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D, dtype=torch.float64)
    slip = torch.zeros(n, Hq, dtype=torch.float64)
    for i in range(n):
        s = seen[i]
        if not bool(s.any()):
            continue
        x = torch.einsum("hd,jhd->hj", q[i], k[s]) * scale
        w = torch.softmax(x, -1)
        o[i] = torch.einsum("hj,jhd->hd", w, v[s])
        size[i] = torch.einsum("hj,jhd->hd", w, v[s].abs())
        terms = torch.einsum("hd,jhd->hj", q[i].abs(), k[s].abs()).amax(-1) * abs(scale)
        slip[i] = (D + 4) * 2.0**-24 * terms
    return o, size, slip


def attend_bound(o, size, slip, dtype, m):
    """|error| of an output. Its own rounding, half a step. Of its terms' sizes: each weight's rounding to bf16 (half a step)
    where the inputs are bf16; the scores' rounding (a sum of D products and the products by scale and by log2 e), in a weight
    and in their sum; exponentials (2 of 2^-24), sums of m weights and of m products, of both 2^-24 a term."""
    c = 2 * slip[..., None] + (2 * m + 16) * 2.0**-24 + (half_step(dtype) if dtype == torch.bfloat16 else 0.0)
    return half_step(dtype) * (o.abs() + c * size) + c * size


def within(got, want, bound) -> float:
    """The largest |got - want| / bound (NaN anywhere: infinite)."""
    d = (got.detach().cpu().double() - want).abs() / bound.clamp_min(1e-300)
    return math.inf if bool(torch.isnan(d).any()) else float(d.max()) if d.numel() else 0.0

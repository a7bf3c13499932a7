"""Plain float64 statements of linear attention and of the projection with an epilogue, and the bounds of their kernels."""

from __future__ import annotations

import math

import torch


def inputs(lead, Hk, Hv, K, V, seed, dtype=torch.bfloat16, n_states=0, slow=1.0, resets=0.0):
    """q, k (unit rows), v, g (log decays a token and head, from fast to slow heads), s0 -- on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k = (torch.nn.functional.normalize(r(*lead, Hk, K), dim=-1).to(dtype) for _ in range(2))
    v = r(*lead, Hv, V).to(dtype)
    rate = 0.7 * 2.0 ** (-6.0 * torch.arange(Hv) / max(Hv - 1, 1)) * slow
    g = -rate * 2 * torch.sigmoid(r(*lead, Hv))
    if resets:
        g = torch.where(torch.rand(*lead, 1, generator=gen) < resets, torch.full((), -math.inf), g)
    s0 = 0.5 * r(n_states, Hv, V, K) if n_states else None
    return {"q": q, "k": k, "v": v, "g": g, "s0": s0}


def tokens(q, k, v, g, s0=None, scale=None, cu=None):
    """The recurrence token by token in float64: (o, final states, and both with every value's absolute value in its
    place: the sizes that rounding errors go by). [B, T, ...] batches, or B = 1 with the bounds ``cu``."""
    q, k, v, g = (t.double().cpu() for t in (q, k, v, g))
    B, T, Hv, V = v.shape
    Hk, K = q.shape[2:]
    g = g.expand(B, T, Hv)
    q, k = (t.repeat_interleave(Hv // Hk, 2) for t in (q, k))
    q = q * (K**-0.5 if scale is None else scale)
    runs = [(b, 0, T) for b in range(B)] if cu is None else [(0, a, e) for a, e in zip(cu, cu[1:])]
    o, mag = torch.zeros(B, T, Hv, V, dtype=torch.float64), torch.zeros(B, T, Hv, V, dtype=torch.float64)
    out, out_mag = [], []
    for i, (b, lo, hi) in enumerate(runs):
        s = torch.zeros(Hv, V, K, dtype=torch.float64) if s0 is None else s0[i].double().cpu().clone()
        m = s.abs()
        for t in range(lo, hi):
            a = torch.exp(g[b, t])[:, None, None]
            u = v[b, t][:, :, None] * k[b, t][:, None, :]
            s, m = a * s + u, a * m + u.abs()
            o[b, t] = (s @ q[b, t][:, :, None])[..., 0]
            mag[b, t] = (m @ q[b, t].abs()[:, :, None])[..., 0]
        out.append(s)
        out_mag.append(m)
    return o, torch.stack(out), mag, torch.stack(out_mag)


def out_bound(o, mag, dtype, T, K):
    """|error| of an output. Its own rounding: half a step, eps / 2 of its value. The rest goes by the sum of its terms'
    sizes: fp32 sums, of K products in q . k, of at most 128 tokens of a segment, of K products with the state and of T
    tokens in the state, 2^-24 each; exponents, sums of at most 128 log decays that carry 2^-24 of their size a level of
    a scan and whose terms are smaller by their exponential (x exp(-x) < 1/2): 64 steps; and, for bf16 inputs, P and the
    state as two bf16 terms, each off by 2^-8 of what it stands for: 2^-16."""
    c = (2 * K + 128 + T + 64) * 2.0**-24 + (2.0**-16 if dtype == torch.bfloat16 else 0.0)
    return torch.finfo(dtype).eps / 2 * (o.abs() + c * mag) + c * mag


def state_bound(mag, T):
    """|error| of a state (fp32): sums over T tokens, decays as above, weighted values in three bf16 terms (2^-24)."""
    return (T + 64 + 2) * 2.0**-24 * mag


def within(got, want, bound) -> float:
    """The largest |got - want| / bound (NaN anywhere: infinite)."""
    d = (got.detach().cpu().double() - want).abs() / bound.clamp_min(1e-300)
    return math.inf if bool(torch.isnan(d).any()) else float(d.max()) if d.numel() else 0.0

"""Values that show single keys: of each key at most one column is not zero, and no column is of many keys, so that an output's
bound (``attn_testing.attend_bound``, which goes by the sizes of its terms) is a small part of what one key adds to it."""

from __future__ import annotations

import torch

import attn_testing as A

EVERY = 16  # one key of each run of as many has a value: one at least of each of the kernels' tiles


def planted(n, Hk, D, dtype, also=()):
    """(v [n, Hk, D], keys with a value, their columns for key head 0; for head h the columns are h further). The place of the
    key goes from run to run. `also`: keys that have one besides (the ends of windows, chunks, sinks)."""
    t = torch.arange(-(-n // EVERY))
    keys = torch.unique(torch.cat([t * EVERY + (7 * t) % EVERY, torch.tensor([0, n - 1, *also], dtype=torch.long)]))
    keys = keys[(keys >= 0) & (keys < n)]
    rank = torch.arange(len(keys))
    v = torch.zeros(n, Hk, D)
    for h in range(Hk):
        v[keys, h, (rank + h) % D] = 1 + 0.25 * (rank // D % 3)  # (exact in bf16)
    return v.to(dtype), keys, rank % D


def queries_and_keys(g, lead_q, lead_k, Hq, Hk, D, dtype):
    """Scores of a quarter: weights within some factor of two of one another."""
    return (0.25 * A.randn(g, *lead_q, Hq, D)).to(dtype), A.randn(g, *lead_k, Hk, D, dtype=dtype)


def least_mistake(q, k, v, keys, columns, p, window, sinks, dtype):
    """One row q [Hq, D] at position p: the least that a mistake with one planted key (a seen one lost, a seen one taken twice,
    one taken that is not seen) is off by, in bounds, over all query heads."""
    n, Hk, D = k.shape
    Hq = q.shape[0]
    want, size, slip = A.attend(q[None], k, v, torch.tensor([p]), window=window, sinks=sinks)
    bound = A.attend_bound(want, size, slip, dtype, n)[0]
    k64, v64 = (x.double().repeat_interleave(Hq // Hk, 1) for x in (k, v))
    j = torch.arange(n)
    seen = (j <= p) & ((p - j < window) | (j < sinks)) if window is not None else j <= p
    w = torch.exp(torch.matmul(q.double()[:, None], k64.permute(1, 2, 0))[:, 0] * D**-0.5)  # [Hq, n]
    total = (w * seen).sum(-1, keepdim=True)
    h = torch.arange(Hq)[:, None]
    column = (columns[None] + h // (Hq // Hk)) % D  # [Hq, planted]
    part, weight = w[:, keys] * v64[keys[None], h, column], w[:, keys]
    o, b = want[0].gather(1, column), bound.gather(1, column)
    lost = (o * total - part) / (total - weight)
    more = (o * total + part) / (total + weight)
    # (an output of a column without seen keys has no bound above 0: any part of one is a mistake)
    off = torch.where(seen[keys], torch.minimum((lost - o).abs(), (more - o).abs()), (more - o).abs())
    return float((off / b.clamp_min(1e-300)).min())

"""The attention sublayer that stands between gated-delta-rule layers, as measurable cases.

Three operators, each through its public entry point:

* ``rope``  norms of queries and keys for each head with the position rotation, keys and values written into a cache
  (``qk_norm_rope``);
* ``attn``  causal attention over whole sequences with a sliding window and a few first tokens that stay visible
  (``window_attn_fwd``);
* ``step``  the same for one token of each of B streams, over a paged cache (``window_attn_step``).

A query at position p sees key j where ``j <= p`` and (``p - j < window`` or ``j < sinks``); window 0 stands for none. A row
that sees nothing is zero. The last query of a sequence stands at the sequence's last key.
"""

from __future__ import annotations

import importlib
import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST_ATTN = 16384 * 16384 // 2 * 16 * 128  # visible pairs x heads x head size of the largest listed prompt
MOST_CACHE = 64 * 8192 * 4 * 128  # elements of the largest listed K cache
MOST_ROPE = 30526 * 18 * 128  # elements of q and k of the largest listed rows
PAGE = 64


def listed():
    return [
        # one stream's token: latency counts
        {"name": "rope_b1", "kind": "rope", "rows": 1, "Hq": 8, "Hk": 2, "D": 128, "rot": 128, "pairs": "halves",
         "weights": True, "cache": True, "far": 4096, "dtype": "bf16"},
        # a decode batch, partly rotated heads, into the cache
        {"name": "rope_b64", "kind": "rope", "rows": 64, "Hq": 16, "Hk": 4, "D": 64, "rot": 32, "pairs": "adjacent",
         "weights": True, "cache": True, "far": 1 << 20, "dtype": "f32"},
        # a server's packed prompts, as many rows as the packed prefill benchmark has
        {"name": "rope_t30526", "kind": "rope", "rows": 30526, "Hq": 16, "Hk": 2, "D": 128, "rot": 128, "pairs": "halves",
         "weights": True, "cache": False, "far": 32768, "dtype": "bf16"},
        # two requests' first window of 64 rows
        {"name": "attn_b2_t64", "kind": "attn", "n": 2, "lo": 64, "hi": 64, "past": 0, "pick": 0, "packed": False, "Hq": 8,
         "Hk": 2, "D": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # one prompt in 32 bits, an odd length, a window with sinks
        {"name": "attn_t1000_f32", "kind": "attn", "n": 1, "lo": 1000, "hi": 1000, "past": 0, "pick": 0, "packed": False,
         "Hq": 4, "Hk": 4, "D": 64, "window": 256, "sinks": 4, "dtype": "f32"},
        # a server's batch of prompts of every length up to 2048, packed, behind what earlier calls left of each
        {"name": "attn_packed_n32", "kind": "attn", "n": 32, "lo": 1, "hi": 2048, "past": 512, "pick": 7, "packed": True,
         "Hq": 16, "Hk": 4, "D": 128, "window": 512, "sinks": 4, "dtype": "bf16"},
        # the context's whole length through a window
        {"name": "attn_t32768_w1024", "kind": "attn", "n": 1, "lo": 32768, "hi": 32768, "past": 0, "pick": 0,
         "packed": False, "Hq": 16, "Hk": 4, "D": 128, "window": 1024, "sinks": 4, "dtype": "bf16"},
        # a long prompt without a window
        {"name": "attn_t16384", "kind": "attn", "n": 1, "lo": 16384, "hi": 16384, "past": 0, "pick": 0, "packed": False,
         "Hq": 16, "Hk": 4, "D": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # two streams of the serving layer's smallest graph, a short cache
        {"name": "step_b2_l700", "kind": "step", "B": 2, "lo": 650, "hi": 700, "pick": 0, "room": 1024, "paged": True,
         "Hq": 8, "Hk": 2, "D": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # one stream at the context's end: few rows, a long axis
        {"name": "step_b1_l32768", "kind": "step", "B": 1, "lo": 32768, "hi": 32768, "pick": 0, "room": 32768,
         "paged": True, "Hq": 16, "Hk": 4, "D": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a batch behind a window, in 32 bits, a cache of one run of rows a stream
        {"name": "step_b48_w600", "kind": "step", "B": 48, "lo": 1, "hi": 4000, "pick": 3, "room": 4096, "paged": False,
         "Hq": 8, "Hk": 8, "D": 64, "window": 600, "sinks": 5, "dtype": "f32"},
        # a full decode batch over long caches
        {"name": "step_b64_l8192", "kind": "step", "B": 64, "lo": 4096, "hi": 8192, "pick": 5, "room": 8192, "paged": True,
         "Hq": 16, "Hk": 4, "D": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "step", "step"])
    D = rng.choice([64, 128, 128])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 4, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "rope":
        return {"kind": kind, "rows": _log(rng, 1, min(30526, MOST_ROPE // ((hq + hk) * D))), "Hq": hq, "Hk": hk, "D": D,
                "rot": rng.choice([D, D, D // 2, 16]), "pairs": rng.choice(["halves", "halves", "adjacent"]),
                "weights": rng.random() < 0.7, "cache": rng.random() < 0.5, "far": _log(rng, 1024, 1 << 20), "dtype": dtype}
    window = rng.choice([0, _log(rng, 1, 4096), _log(rng, 64, 2048)])
    sinks = rng.choice([0, 4, rng.randint(1, 130)])
    if kind == "attn":
        n = _log(rng, 1, 32)
        hi = _log(rng, 1, 16384)
        past = rng.choice([0, 0, _log(rng, 1, 4096)])
        packed = n > 1 and rng.random() < 0.6
        share = 1 if dtype == "bf16" else 8
        while n * hi * (past + (hi // 2 if window == 0 else min(hi // 2, window))) * hq * D * share > MOST_ATTN \
                or n * (hi + past) > 65536:
            hi = max(1, hi * 3 // 4)
            n = max(1, n * 3 // 4)
            past = past * 3 // 4
        return {"kind": kind, "n": n, "lo": rng.randint(1, hi) if packed else hi, "hi": hi, "past": past,
                "pick": rng.randrange(10**6), "packed": packed and n > 1, "Hq": hq, "Hk": hk, "D": D, "window": window,
                "sinks": sinks, "dtype": dtype}
    B = _log(rng, 1, 256)
    most = MOST_CACHE // (B * hk * D * (1 if dtype == "bf16" else 2))
    hi = _log(rng, 1, max(1, min(32768, most)))
    return {"kind": kind, "B": B, "lo": rng.randint(0, hi), "hi": hi, "pick": rng.randrange(10**6),
            "room": -(-hi // PAGE) * PAGE, "paged": rng.random() < 0.6, "Hq": hq, "Hk": hk, "D": D, "window": window,
            "sinks": sinks, "dtype": dtype}


# ------------------------------------------------------------------------------------------------- inputs


def _numbers(pick, n, lo, hi):
    g = torch.Generator().manual_seed(pick)
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def _lengths(c):
    """(queries, keys) of each sequence of a prompt case."""
    q = _numbers(c["pick"], c["n"], c["lo"], c["hi"]) if c["packed"] else [c["hi"]] * c["n"]
    past = _numbers(c["pick"] + 1, c["n"], 0, c["past"]) if c["packed"] else [c["past"]] * c["n"]
    return q, [a + b for a, b in zip(q, past)]


class _Rand:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def __call__(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float32).to(dtype)

    def rank(self, n):
        return torch.argsort(torch.rand(n, generator=self.gen, device="cuda"))

    def below(self, n, top):
        return torch.randint(0, top, (n,), generator=self.gen, device="cuda")


def _unit(x):
    """Rows of root mean square 1, as a norm without weights leaves them."""
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def _bounds(lengths):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, r = SimpleNamespace(**case), _Rand(seed)
    dt = DTYPES[c.dtype]
    if c.kind == "rope":
        # q, k and v as slices of one projection's rows
        proj = r(c.rows, (c.Hq + 2 * c.Hk) * c.D, dtype=dt)
        q, k, v = proj.split([c.Hq * c.D, c.Hk * c.D, c.Hk * c.D], -1)
        s = SimpleNamespace(c=c, q=q.unflatten(-1, (c.Hq, c.D)), k=k.unflatten(-1, (c.Hk, c.D)),
                            v=v.unflatten(-1, (c.Hk, c.D)), positions=r.below(c.rows, c.far), qw=None, kw=None, cache=None)
        s.inv_freq = 10000.0 ** (-torch.arange(0, c.rot, 2, dtype=torch.float64, device="cuda") / c.rot)
        if c.weights:
            s.qw, s.kw = (1 + 0.1 * r(c.D)).to(dt), (1 + 0.1 * r(c.D)).to(dt)
        if c.cache:
            pages = -(-c.rows // PAGE) + 3
            s.cache = [torch.zeros(pages, PAGE, c.Hk, c.D, dtype=dt, device="cuda") for _ in range(2)]
            s.rows = r.rank(pages * PAGE)[: c.rows].contiguous()
        return s
    s = SimpleNamespace(c=c, scale=c.D**-0.5)
    if c.kind == "attn":
        s.nq, s.nk = _lengths(case)
        lead_q, lead_k = ((1, sum(s.nq)), (1, sum(s.nk))) if c.packed else ((c.n, c.hi), (c.n, c.hi + c.past))
        s.q, s.k = _unit(r(*lead_q, c.Hq, c.D)).to(dt), _unit(r(*lead_k, c.Hk, c.D)).to(dt)
        s.v = r(*lead_k, c.Hk, c.D, dtype=dt)
        s.cu, s.cu_k = (_bounds(s.nq), _bounds(s.nk)) if c.packed else (None, None)
        return s
    s.q = _unit(r(c.B, c.Hq, c.D)).to(dt)
    lengths = _numbers(c.pick, c.B, c.lo, c.hi)
    s.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s.pages = None
    if c.paged:
        each = c.room // PAGE
        shape = (c.B * each + 3, PAGE)
        s.pages = r.rank(shape[0])[: c.B * each].view(c.B, each).int()
    else:
        shape = (c.B, c.room)
    s.kc, s.vc = _unit(r(*shape, c.Hk, c.D)).to(dt), r(*shape, c.Hk, c.D, dtype=dt)
    return s


# ---------------------------------------------------------------------------------------------- plain forms


def _plain_rope(s):
    c = s.c
    angle = s.positions.double()[:, None] * s.inv_freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        if w is not None:
            x = x * w.float()
        x, rest = x[..., : c.rot], x[..., c.rot:]
        if c.pairs == "halves":
            a, b = x[..., : c.rot // 2], x[..., c.rot // 2:]
            x = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = x[..., 0::2], x[..., 1::2]
            x = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([x, rest], -1).to(DTYPES[c.dtype])

    q, k = turn(s.q, s.qw), turn(s.k, s.kw)
    if s.cache is None:
        return q, k
    for cache, x in zip(s.cache, (k, s.v)):
        cache.view(-1, c.Hk, c.D)[s.rows] = x
    return q, s.cache[0], s.cache[1]


def _softmax_rows(scores, seen):
    """Weights of the last axis where ``seen``, zeros in rows that see nothing."""
    scores = torch.where(seen, scores, torch.full((), -math.inf, device="cuda"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attend(s, q, k, v):
    """One sequence: q [nq, Hq, D], k, v [nk, Hk, D], by blocks of queries and the keys that a block may see."""
    c = s.c
    nq, nk = q.shape[0], k.shape[0]
    out, block = [], 512
    for a in range(0, nq, block):
        b = min(nq, a + block)
        first, last = nk - nq + a, nk - nq + b  # the block's positions
        lo = max(0, first - c.window + 1) if c.window else 0
        js = torch.arange(lo, max(last, lo), device="cuda")
        if c.window and c.sinks:
            js = torch.cat([torch.arange(min(c.sinks, lo), device="cuda"), js])
        ps = torch.arange(first, last, device="cuda")[:, None]
        seen = js <= ps
        if c.window:
            seen = seen & ((ps - js < c.window) | (js < c.sinks))
        kk, vv = (x[js].float().transpose(0, 1) for x in (k, v))  # [Hk, keys, D]
        qq = q[a:b].float().unflatten(1, (c.Hk, -1)).permute(1, 2, 0, 3).flatten(1, 2)  # [Hk, G * rows, D]
        w = _softmax_rows((qq @ kk.transpose(1, 2) * s.scale).unflatten(1, (-1, b - a)), seen)
        o = w.flatten(1, 2) @ vv
        out.append(o.unflatten(1, (-1, b - a)).permute(2, 0, 1, 3).flatten(1, 2))
    return torch.cat(out)


def _plain_attn(s):
    q, k, v = ((x[0].split(n) if s.c.packed else x) for x, n in ((s.q, s.nq), (s.k, s.nk), (s.v, s.nk)))
    o = [_plain_attend(s, *x) for x in zip(q, k, v)]
    return (torch.cat(o).unsqueeze(0) if s.c.packed else torch.stack(o)).to(s.q.dtype)


def _step_rows(s):
    """Rows of the flat cache that hold each stream's positions, [B, room]."""
    p = torch.arange(s.c.room, device="cuda")
    if s.pages is None:
        return torch.arange(s.c.B, device="cuda")[:, None] * s.c.room + p
    return s.pages.long()[:, p // PAGE] * PAGE + p % PAGE


def _step_seen(s):
    j, n = torch.arange(s.c.room, device="cuda"), s.lengths.long()[:, None]
    seen = j < n
    return seen & ((n - 1 - j < s.c.window) | (j < s.c.sinks)) if s.c.window else seen


def _plain_step(s):
    c, rows = s.c, _step_rows(s)
    seen = _step_seen(s)
    out = []
    for b in range(0, c.B, 16):  # some streams at a time
        k, v = (x.view(-1, c.Hk, c.D)[rows[b: b + 16]].float().transpose(1, 2) for x in (s.kc, s.vc))  # [b, Hk, room, D]
        q = s.q[b: b + 16].float().unflatten(1, (c.Hk, -1))
        w = _softmax_rows(q @ k.transpose(-1, -2) * s.scale, seen[b: b + 16, None, None])
        out.append((w @ v).flatten(1, 2))
    return torch.cat(out).to(s.q.dtype)


def run(state):
    s = state
    if own:
        ops = importlib.import_module("zonos3-mini_amd").ops
        if s.c.kind == "rope":
            adjacent = s.c.pairs == "adjacent"
            if s.cache is None:
                return ops.qk_norm_rope(s.q, s.k, s.positions, s.inv_freq, s.qw, s.kw, interleaved=adjacent)
            q, _ = ops.qk_norm_rope(s.q, s.k, s.positions, s.inv_freq, s.qw, s.kw, interleaved=adjacent, v=s.v,
                                    k_cache=s.cache[0], v_cache=s.cache[1], rows=s.rows, output_k=False)
            return q, s.cache[0], s.cache[1]
        window = s.c.window or None
        if s.c.kind == "attn":
            return ops.window_attn_fwd(s.q, s.k, s.v, window=window, sinks=s.c.sinks, cu_seqlens=s.cu, cu_seqlens_k=s.cu_k)
        return ops.window_attn_step(s.q, s.kc, s.vc, s.lengths, window=window, sinks=s.c.sinks, pages=s.pages)
    if s.c.kind == "rope":
        return _plain_rope(s)
    return _plain_attn(s) if s.c.kind == "attn" else _plain_step(s)


def _visible(n, window, sinks):
    """Keys that the query at position n - 1 sees."""
    if n <= 0:
        return 0
    return n if not window else min(n, window) + min(sinks, max(0, n - window))


def _visible_upto(n, window, sinks):
    """The sum of ``_visible`` over the positions 0 .. n - 1."""
    n = max(n, 0)
    if not window or n <= window:
        return n * (n + 1) // 2
    far = n - window  # positions that the window leaves the start of the sequence behind at
    reach = min(far, sinks)
    return window * (window + 1) // 2 + far * window + reach * (reach + 1) // 2 + (far - reach) * sinks


def work(case):
    c = SimpleNamespace(**case)
    size = 2 if c.dtype == "bf16" else 4
    if c.kind == "rope":
        n = 2 * c.rows * (c.Hq + c.Hk) * c.D * size + c.rows * 8 + c.rot * 4
        if c.cache:
            n += 2 * c.rows * c.Hk * c.D * size + c.rows * 8
        return {"bytes": n, "flops": c.rows * (c.Hq + c.Hk) * (4 * c.D + 3 * c.rot)}
    if c.kind == "attn":
        nq, nk = _lengths(case)
        pairs = sum(_visible_upto(b, c.window, c.sinks) - _visible_upto(b - a, c.window, c.sinks) for a, b in zip(nq, nk))
        used = sum(b if not c.window else min(b, a + c.window - 1 + min(c.sinks, max(0, b - a - c.window + 1)))
                   for a, b in zip(nq, nk))
        return {"bytes": size * c.D * (2 * sum(nq) * c.Hq + 2 * used * c.Hk), "flops": 4 * pairs * c.Hq * c.D}
    seen = sum(_visible(n, c.window, c.sinks) for n in _numbers(c.pick, c.B, c.lo, c.hi))
    return {"bytes": size * c.D * (2 * seen * c.Hk + 2 * c.B * c.Hq), "flops": 4 * seen * c.Hq * c.D}


# ---------------------------------------------------------------------------------------------------- exact


def _exact_rope(s):
    c = s.c
    turns = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s.positions.double()[:, None] * s.inv_freq)

    def each(x, w):
        x = x.double()
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c.D + 1e-6)
        x = x if w is None else x * w.double()
        out = x.clone()
        half = c.rot // 2
        a, b = (slice(0, half), slice(half, c.rot)) if c.pairs == "halves" else (slice(0, c.rot, 2), slice(1, c.rot, 2))
        z = torch.complex(x[..., a], x[..., b]) * turns[:, None]
        out[..., a], out[..., b] = z.real, z.imag
        return out

    q, k = each(s.q, s.qw), each(s.k, s.kw)
    if s.cache is None:
        return q, k
    kc, vc = (x.double().flatten(0, 1) for x in s.cache)
    kc[s.rows], vc[s.rows] = k, s.v.double()
    return q, kc.view(s.cache[0].shape), vc.view(s.cache[1].shape)


def _exact_one(q, k, v, p, js, window, sinks, scale):
    """One key head: queries q [n, G, D] at positions p [n], all of its keys k and values v at positions js."""
    ok = p[:, None] >= js
    if window:
        ok &= (p[:, None] < js + window) | (js < sinks)
    a = torch.matmul(q.flatten(0, 1), k.T).view(q.shape[0], q.shape[1], -1) * scale
    a = a.masked_fill(~ok[:, None], -math.inf).softmax(-1).masked_fill(~ok.any(-1)[:, None, None], 0.0)
    return torch.matmul(a.flatten(0, 1), v).view(q.shape)


def exact(case, seed):
    s = prepare(case, seed)
    c = s.c
    if c.kind == "rope":
        return _exact_rope(s)
    G = c.Hq // c.Hk
    if c.kind == "step":
        o = torch.zeros(c.B, c.Hq, c.D, dtype=torch.float64, device="cuda")
        rows = _step_rows(s)
        for b, n in enumerate(s.lengths.tolist()):
            k, v = (x.view(-1, c.Hk, c.D)[rows[b, :n]].double() for x in (s.kc, s.vc))
            p, js = torch.tensor([n - 1], device="cuda"), torch.arange(n, device="cuda")
            for h in range(c.Hk):
                if n:
                    o[b, h * G: (h + 1) * G] = _exact_one(s.q[b: b + 1, h * G: (h + 1) * G].double(), k[:, h], v[:, h], p, js,
                                                          c.window, c.sinks, s.scale)[0]
        return o
    o = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for i, (nq, nk) in enumerate(zip(s.nq, s.nk)):
        at = (0, slice(q0, q0 + nq)) if c.packed else (i, slice(None))
        keys = (0, slice(k0, k0 + nk)) if c.packed else (i, slice(None))
        q, k, v, js = s.q[at].double(), s.k[keys].double(), s.v[keys].double(), torch.arange(nk, device="cuda")
        p = js[-nq:]
        for h in range(c.Hk):
            for a in range(0, nq, 2048):
                o[at][a: a + 2048, h * G: (h + 1) * G] = _exact_one(q[a: a + 2048, h * G: (h + 1) * G], k[:, h], v[:, h],
                                                                    p[a: a + 2048], js, c.window, c.sinks, s.scale)
        q0, k0 = q0 + nq, k0 + nk
    return o

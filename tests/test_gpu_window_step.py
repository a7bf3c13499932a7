"""Single-token attention over a cache against float64 (bounds: ``attn_testing``)."""

from __future__ import annotations

import pytest
import torch

import attn_testing as A
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def _cache(lengths, page, Hq, Hk, D, seed, dtype, dense=False, spare=2):
    """q, caches whose rows outside the streams hold NaN, pages in any order, and each stream's own k and v."""
    g = torch.Generator().manual_seed(seed)
    B, most = len(lengths), max(max(lengths), 1)
    each = 1 if dense else -(-most // page) + 1
    shape = (B, most + 3) if dense else (B * each + spare, page)
    kc, vc = (torch.full((*shape, Hk, D), NAN, dtype=dtype) for _ in range(2))
    pages = torch.arange(B)[:, None] if dense else torch.randperm(shape[0], generator=g)[: B * each].view(B, each)
    ks, vs = [], []
    for b, n in enumerate(lengths):
        k, v = A.randn(g, n, Hk, D, dtype=dtype), A.randn(g, n, Hk, D, dtype=dtype)
        p = torch.arange(n)
        row = pages[b, p // shape[1]] * shape[1] + p % shape[1]
        kc.view(-1, Hk, D)[row], vc.view(-1, Hk, D)[row] = k, v
        ks.append(k)
        vs.append(v)
    q = A.randn(g, B, Hq, D, dtype=dtype)
    return q, kc, vc, (None if dense else pages.int()), ks, vs


def _hold(o, q, ks, vs, dtype, **kw):
    for b, (k, v) in enumerate(zip(ks, vs)):
        n = k.shape[0]
        want = A.attend(q[b: b + 1], k, v, torch.tensor([n - 1]), **kw)
        e = A.within(o[b: b + 1], want[0], A.attend_bound(*want, dtype, n))
        assert e <= 1, (b, n, e)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [None, 1, 4, 16, 64, 512])
@pytest.mark.parametrize("Hq,Hk,D,window,sinks", [(8, 2, 128, None, 0), (3, 3, 64, 70, 5), (20, 1, 64, 33, 40), (17, 1, 128, 1, 0)])
def test_against_float64(gdn, cuda, Hq, Hk, D, window, sinks, page, dtype):
    announce(f"window_attn_step {Hq}/{Hk} D {D} window {window} sinks {sinks} page {page} {dtype}")
    lengths = [1, 700, 0, 33, 64, 333]
    q, kc, vc, pages, ks, vs = _cache(lengths, page or 1, Hq, Hk, D, 31, dtype, dense=page is None)
    o = gdn.window_attn_step(q.to(cuda), kc.to(cuda), vc.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
                             window=window, sinks=sinks, pages=None if pages is None else pages.to(cuda))
    torch.cuda.synchronize()
    assert o.shape == q.shape and o.dtype == dtype
    _hold(o, q, ks, vs, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,longest,window,sinks", [(1, 20000, None, 0), (70, 300, None, 0), (9, 9000, 2000, 4)])
def test_long_and_many(gdn, cuda, B, longest, window, sinks, dtype):
    """One stream over many chunks, many streams, and chunks that a window leaves unused."""
    announce(f"window_attn_step {B} up to {longest} window {window} {dtype}")
    lengths = [max(1, longest - 257 * b) for b in range(B)]
    q, kc, vc, pages, ks, vs = _cache(lengths, 64, 4, 2, 128, 32, dtype)
    o = gdn.window_attn_step(q.to(cuda), kc.to(cuda), vc.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
                             window=window, sinks=sinks, pages=pages.to(cuda))
    torch.cuda.synchronize()
    _hold(o, q, ks, vs, dtype, window=window, sinks=sinks)


def test_slices_of_a_joint_cache(gdn, cuda):
    announce("window_attn_step joint cache, projection rows")
    q, kc, vc, pages, ks, vs = _cache([90, 41], 16, 4, 2, 64, 33, BF)
    joint = torch.stack([kc, vc], 2).to(cuda)
    wide = torch.cat([q.flatten(1), q.flatten(1)], -1).to(cuda)
    o = gdn.window_attn_step(wide[:, 256:].unflatten(-1, (4, 64)), joint[:, :, 0], joint[:, :, 1],
                             torch.tensor([90, 41], dtype=torch.int32, device=cuda), pages=pages.to(cuda), scale=0.5)
    torch.cuda.synchronize()
    _hold(o, q, ks, vs, BF, scale=0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_and_pages_out_of_range(gdn, cuda, dtype):
    """Lengths below zero and past the pages are clamped; a page that is not in the cache is not seen, and neither are pages
    behind a window's start."""
    announce(f"window_attn_step out of range {dtype}")
    q, kc, vc, pages, ks, vs = _cache([200, 200, 200, 200], 16, 4, 2, 64, 34, dtype)
    pages = pages[:, :12]  # (192 positions)
    pages[2, 3], pages[2, 5] = -1, 1 << 30
    pages[3] = -5
    lengths = torch.tensor([-3, 1000, 192, 192], dtype=torch.int32)
    args = [t.to(cuda) for t in (q, kc, vc, lengths)]
    o = gdn.window_attn_step(*args, pages=pages.to(cuda)).cpu()
    torch.cuda.synchronize()
    assert not bool(o[0].any()) and not bool(o[3].any())
    _hold(o[1:2], q[1:2], [ks[1][:192]], [vs[1][:192]], dtype)
    there = [p for p in range(192) if p // 16 not in (3, 5)]
    _hold(o[2:3], q[2:3], [ks[2][there]], [vs[2][there]], dtype)
    o = gdn.window_attn_step(*args, window=90, pages=pages.to(cuda)).cpu()
    _hold(o[2:3], q[2:3], [ks[2][:192]], [vs[2][:192]], dtype, window=90)


def test_step_and_prompt_agree(gdn, cuda):
    """The sublayer as it is used: a prompt through norms, rotation, cache and attention, then tokens one at a time, against
    the same tokens as one prompt."""
    announce("attention sublayer, prompt then steps")
    B, T, more, Hq, Hk, D, page, window, sinks = 2, 75, 40, 8, 2, 64, 16, 50, 3
    g = torch.Generator().manual_seed(35)
    total = T + more
    proj = A.randn(g, B, total, (Hq + 2 * Hk) * D, dtype=BF).to(cuda)
    freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).to(cuda)
    qw, kw = ((1 + 0.1 * A.randn(g, D)).to(cuda) for _ in range(2))
    each = -(-total // page)
    pages = torch.randperm(B * each, generator=g).view(B, each).int().to(cuda)
    kc, vc = (torch.full((B * each, page, Hk, D), NAN, dtype=BF, device=cuda) for _ in range(2))

    def parts(x):
        return [t.unflatten(-1, (-1, D)) for t in x.split([Hq * D, Hk * D, Hk * D], -1)]

    def rows(p):
        return (pages[:, p // page].long() * page + p % page).contiguous()

    p = torch.arange(total, device=cuda)
    at = p.expand(B, total).contiguous()
    q, k, v = parts(proj)
    q_all, k_all = gdn.qk_norm_rope(q, k, at, freq, qw, kw)
    whole = gdn.window_attn_fwd(q_all, k_all, v, window=window, sinks=sinks)

    q, k, v = parts(proj[:, :T])
    qn, kn = gdn.qk_norm_rope(q, k, at[:, :T].contiguous(), freq, qw, kw, v=v, k_cache=kc, v_cache=vc, rows=rows(p[:T]))
    out = [gdn.window_attn_fwd(qn, kn, v, window=window, sinks=sinks)]
    assert torch.equal(qn, q_all[:, :T]) and torch.equal(kn, k_all[:, :T])
    for t in range(T, total):
        q, k, v = parts(proj[:, t])
        qn, none = gdn.qk_norm_rope(q, k, at[:, t].contiguous(), freq, qw, kw, v=v, k_cache=kc, v_cache=vc, rows=rows(p[t]),
                                    output_k=False)
        assert none is None and torch.equal(qn, q_all[:, t])
        lengths = torch.full((B,), t + 1, dtype=torch.int32, device=cuda)
        out.append(gdn.window_attn_step(qn, kc, vc, lengths, window=window, sinks=sinks, pages=pages).unsqueeze(1))
    torch.cuda.synchronize()
    got = torch.cat(out, 1)
    v = parts(proj)[2]
    for b in range(B):
        want = A.attend(q_all[b], k_all[b], v[b], torch.arange(total), window=window, sinks=sinks)
        bound = A.attend_bound(*want, BF, total)
        assert A.within(got[b], want[0], bound) <= 1 and A.within(whole[b], want[0], bound) <= 1

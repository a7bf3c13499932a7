"""Attention with a window and sinks over whole sequences against float64 (bounds: ``attn_testing``)."""

from __future__ import annotations

import pytest
import torch

import attn_testing as A
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _inputs(B, Tq, Tk, Hq, Hk, D, seed, dtype, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(sharp * A.randn(g, B, Tq, Hq, D)).to(dtype), A.randn(g, B, Tk, Hk, D, dtype=dtype),
            A.randn(g, B, Tk, Hk, D, dtype=dtype)]


def _hold(o, q, k, v, dtype, rows=None, **kw):
    """Rows of one sequence against float64: q, o [n, Hq, D] (all, or some of them), the last at the last key."""
    n, m = q.shape[0], k.shape[0]
    at = torch.arange(n) if rows is None else rows
    want = A.attend(q[at], k, v, m - n + at, **kw)
    e = A.within(o.cpu()[at], want[0], A.attend_bound(*want, dtype, m))
    print(f"[errors] {e:.3f} of the bound")
    assert e <= 1, e


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hk,D,window,sinks", [
    (1, 1, 1, 1, 1, 64, None, 0), (2, 64, 64, 8, 2, 128, None, 0), (3, 33, 33, 3, 1, 64, 1, 0), (1, 130, 130, 5, 1, 128, 17, 3),
    (2, 200, 200, 2, 2, 64, 64, 64), (1, 300, 300, 8, 1, 64, 100, 40), (1, 70, 333, 4, 2, 128, 50, 5),
    (1, 1, 500, 4, 4, 64, None, 0), (2, 100, 40, 6, 2, 64, 30, 2), (1, 9, 0, 2, 1, 64, None, 0), (1, 257, 257, 16, 1, 128, 1000, 9),
    (1, 96, 700, 7, 7, 128, 128, 200)])
def test_against_float64(gdn, cuda, B, Tq, Tk, Hq, Hk, D, window, sinks, dtype):
    announce(f"window_attn_fwd {B} x {Tq}/{Tk} {Hq}/{Hk} D {D} window {window} sinks {sinks} {dtype}")
    q, k, v = _inputs(B, Tq, Tk, Hq, Hk, D, Tq + Tk, dtype)
    o = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert o.shape == q.shape and o.dtype == dtype
    for b in range(B):
        _hold(o[b], q[b], k[b], v[b], dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Hq,Hk,D,window,sinks", [(5000, 8, 2, 128, None, 0), (9000, 16, 8, 64, 700, 4),
                                                    (2500, 24, 8, 128, 1100, 70)])
def test_many_tiles(gdn, cuda, T, Hq, Hk, D, window, sinks, dtype):
    """Each of the workgroup sizes, with rows from all over the sequence; scores of up to some twenty."""
    announce(f"window_attn_fwd {T} {Hq}/{Hk} D {D} window {window} sinks {sinks} {dtype}")
    q, k, v = _inputs(1, T, T, Hq, Hk, D, T, dtype, sharp=4.0)
    o = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), window=window, sinks=sinks)
    torch.cuda.synchronize()
    rows = torch.cat([torch.arange(3), torch.randperm(T, generator=torch.Generator().manual_seed(1))[:40],
                      torch.arange(T - 3, T)])
    _hold(o[0], q[0], k[0], v[0], dtype, rows=rows, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,Hk,D,window,sinks", [(4, 2, 64, 40, 3), (8, 1, 128, None, 0)])
@pytest.mark.parametrize("host", [False, True])
def test_packed(gdn, cuda, Hq, Hk, D, window, sinks, host, dtype):
    """Packed sequences, empty ones among them, more queries than keys and fewer; rows behind the last stay as they were."""
    announce(f"window_attn_fwd packed {Hq}/{Hk} D {D} host {host} {dtype}")
    nq, nk = [5, 0, 130, 1, 64, 20, 0, 3], [5, 7, 130, 90, 200, 8, 0, 0]
    Tq, Tk = sum(nq) + (0 if host else 6), sum(nk) + (0 if host else 9)
    q, k, v = _inputs(1, Tq, Tk, Hq, Hk, D, 21, dtype)
    cu, cu_k = (torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32) for n in (nq, nk))
    if not host:  # (rows of no sequence are not read, and what is allocated for them is not written)
        q[:, sum(nq):], k[:, sum(nk):], v[:, sum(nk):] = NAN, NAN, NAN
        keep = torch.full((1, Tq, Hq, D), 7.0, device=cuda, dtype=dtype)
        torch.cuda.synchronize()
        ptr = keep.data_ptr()
        del keep
    o = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), window=window, sinks=sinks,
                            cu_seqlens=cu if host else cu.to(cuda), cu_seqlens_k=cu_k.tolist() if host else cu_k.to(cuda))
    torch.cuda.synchronize()
    if not host and o.data_ptr() == ptr:
        assert bool((o[:, sum(nq):] == 7).all())
    for i in range(len(nq)):
        a, b, c, d = int(cu[i]), int(cu[i + 1]), int(cu_k[i]), int(cu_k[i + 1])
        _hold(o[0, a:b], q[0, a:b], k[0, c:d], v[0, c:d], dtype, window=window, sinks=sinks)


def test_many_packed_sequences(gdn, cuda):
    """More sequences than a wave has lanes, mostly of no or few tokens, and a table's own bounds past the rows."""
    announce("window_attn_fwd 150 packed sequences")
    nq = [(i * 37) % 5 for i in range(149)] + [190]
    cu = torch.tensor([0, *torch.tensor(nq).cumsum(0).tolist()], dtype=torch.int32)
    T = int(cu[-1])
    q, k, v = _inputs(1, T, T, 4, 2, 64, 22, BF)
    past = cu.clone()
    past[-1] += 1000  # (clamped to the rows there are)
    x = [t.to(cuda) for t in (q, k, v)]
    o = gdn.window_attn_fwd(*x, window=60, sinks=2, cu_seqlens=past.to(cuda))
    o2 = gdn.window_attn_fwd(*x, window=60, sinks=2, cu_seqlens=cu.to(cuda))
    torch.cuda.synchronize()
    assert torch.equal(o, o2)
    for i in range(150):
        a, b = int(cu[i]), int(cu[i + 1])
        _hold(o[0, a:b], q[0, a:b], k[0, a:b], v[0, a:b], BF, window=60, sinks=2)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_slices_and_scale(gdn, cuda, dtype):
    announce(f"window_attn_fwd slices {dtype}")
    q, k, v = _inputs(2, 90, 90, 4, 2, 64, 23, dtype)
    wide = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).to(cuda)
    a, b, c = (t.unflatten(-1, (-1, 64)) for t in wide.split([256, 128, 128], -1))
    for scale in (0.3, -0.2, 0.0):
        o = gdn.window_attn_fwd(a, b, c, window=33, sinks=1, scale=scale)
        torch.cuda.synchronize()
        for i in range(2):
            _hold(o[i], q[i], k[i], v[i], dtype, window=33, sinks=1, scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,Hk,D", [(4, 1, 64), (2, 2, 128)])
def test_what_is_not_seen_has_no_part(gdn, cuda, Hq, Hk, D, dtype):
    """Infinities and NaN in keys and values: rows that do not see them are as without them, rows that do are as float64's."""
    announce(f"window_attn_fwd not finite {Hq}/{Hk} D {D} {dtype}")
    T, window, sinks = 300, 70, 3
    q, k, v = _inputs(1, T, T, Hq, Hk, D, 25, dtype)
    clean = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), window=window, sinks=sinks).cpu()
    v[0, 100, 0, 5], v[0, 200, 0, 7], k[0, 250, 0] = INF, NAN, NAN
    o = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), window=window, sinks=sinks).cpu()
    t = torch.arange(T)
    sees = lambda j: (t >= j) & (t - j < window)  # noqa: E731
    heads = torch.arange(Hq) // (Hq // Hk) == 0
    hit = heads[None, :, None] & ((sees(100)[:, None, None] & (torch.arange(D) == 5)) | (sees(200)[:, None, None] & (torch.arange(D) == 7))
                                  | sees(250)[:, None, None].expand(T, 1, D))
    touched = hit.any(-1)
    assert torch.equal(o[0][~touched], clean[0][~touched])  # (rows computed as before)
    e = A.attend(q[0], torch.nan_to_num(k[0].float(), 0, 0, 0), torch.nan_to_num(v[0].float(), 0, 0, 0), t, window=window,
                 sinks=sinks)
    rest = ~hit & ~(heads[None, :, None] & sees(250)[:, None, None]) & touched[..., None]
    zeroed = torch.zeros_like(rest)
    zeroed[:, heads] = (sees(100) | sees(200))[:, None, None]
    free = rest & ~zeroed  # (what a zero in the value's place leaves as it is)
    assert bool(o[0][hit].isnan().any()) and not bool(torch.isfinite(o[0][hit].float()).any())
    other = rest & zeroed
    d = (o[0].double() - e[0]).abs() / A.attend_bound(*e, dtype, T).clamp_min(1e-300)
    assert float(d[other | free].max()) <= 1


def test_scores_beyond_float32(gdn, cuda):
    """Every visible key's score -inf, or one +inf: NaN, as 0 / 0 and inf - inf are; a lone -inf has no weight."""
    announce("window_attn_fwd infinite scores")
    q, k, v = torch.ones(1, 3, 1, 64), torch.ones(1, 3, 1, 64), torch.ones(1, 3, 1, 64)
    k[0, 0, 0, 0] = -INF
    k[0, 2, 0, 0] = INF
    o = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda)).cpu()
    assert bool(o[0, 0].isnan().all()) and bool((o[0, 1] == 1).all()) and bool(o[0, 2].isnan().all())

"""Norms and rotation of queries and keys against float64, and the cache's write (bounds: ``attn_testing``)."""

from __future__ import annotations

import pytest
import torch

import attn_testing as A
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(lead, Hq, Hk, D, R, seed, dtype, far=1 << 16, weights=True):
    g = torch.Generator().manual_seed(seed)
    d = {"q": A.randn(g, *lead, Hq, D, dtype=dtype), "k": A.randn(g, *lead, Hk, D, dtype=dtype),
         "v": A.randn(g, *lead, Hk, D, dtype=dtype), "positions": torch.randint(0, far, lead, generator=g),
         "inv_freq": 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))}
    d["qw"], d["kw"] = ((1 + 0.2 * A.randn(g, D)).to(dtype), (1 + 0.2 * A.randn(g, D)).to(dtype)) if weights else (None, None)
    return d


def _hold(q, k, d, dtype, **kw):
    for name, got, w in (("q", q, d["qw"]), ("k", k, d["kw"])):
        want, bound = A.rope(d[name], d["positions"], d["inv_freq"], w, dtype=dtype, **kw)
        assert got.shape == want.shape and got.dtype == dtype
        e = A.within(got, want, bound)
        print(f"[errors] {name} {e:.3f} of its bound")
        assert e <= 1, (name, e)


def _to(d, cuda):
    return {n: t.to(cuda) if t is not None else None for n, t in d.items()}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,Hq,Hk,D,R,far,weights", [
    ((1,), 8, 2, 128, 128, 1 << 16, True), ((3, 37), 5, 1, 64, 64, 1 << 20, True), ((2, 700), 16, 4, 128, 64, 1 << 20, False),
    ((257,), 3, 3, 64, 16, 32768, True), ((5000,), 40, 8, 128, 128, 1 << 31, True), ((9,), 1, 1, 128, 0, 100, True)])
def test_against_float64(gdn, cuda, lead, Hq, Hk, D, R, far, weights, interleaved, dtype):
    announce(f"qk_norm_rope {lead} {Hq}/{Hk} D {D} R {R} far {far} interleaved {interleaved} {dtype}")
    d = _inputs(lead, Hq, Hk, D, R, 3, dtype, far, weights)
    x = _to(d, cuda)
    q, k = gdn.qk_norm_rope(x["q"], x["k"], x["positions"], x["inv_freq"], x["qw"], x["kw"], interleaved=interleaved)
    torch.cuda.synchronize()
    _hold(q, k, d, dtype, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_slices_types_and_signs(gdn, cuda, dtype):
    """Column slices of a projection, positions of 32 bits and below zero, float32 frequencies and weights, another eps."""
    announce(f"qk_norm_rope slices {dtype}")
    d = _inputs((70,), 6, 2, 64, 32, 5, dtype)
    d["positions"] = torch.arange(70, dtype=torch.int32) - 35
    d["inv_freq"] = d["inv_freq"].float()
    d["qw"], d["kw"] = d["qw"].float(), d["kw"].float()
    wide = torch.cat([d["q"].flatten(1), d["k"].flatten(1), d["v"].flatten(1)], -1).to(cuda)
    q, k, _ = (t.unflatten(-1, (-1, 64)) for t in wide.split([384, 128, 128], -1))
    x = _to(d, cuda)
    assert not q.is_contiguous()
    q, k = gdn.qk_norm_rope(q, k, x["positions"], x["inv_freq"], x["qw"], x["kw"], eps=0.1)
    torch.cuda.synchronize()
    _hold(q, k, d, dtype, eps=0.1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,with_v,output_k", [(1, True, False), (90, True, True), (90, False, False), (3000, True, False)])
def test_cache(gdn, cuda, n, with_v, output_k, dtype):
    """Keys and values at the named rows of slices of a joint cache; every other row, and tokens of rows outside, untouched."""
    announce(f"qk_norm_rope cache {n} v {with_v} k {output_k} {dtype}")
    Hk, D, pages, size = 2, 128, n // 16 + 3, 16
    d = _inputs((n,), 4, Hk, D, 128, 7, dtype)
    x = _to(d, cuda)
    g = torch.Generator().manual_seed(9)
    joint = A.randn(g, pages, size, 2, Hk, D, dtype=dtype).to(cuda)
    before = joint.cpu().clone()
    rows = torch.randperm(pages * size, generator=g)[:n]
    if n > 8:
        rows[3], rows[5], rows[8] = -1, pages * size, 1 << 40
    q, k = gdn.qk_norm_rope(x["q"], x["k"], x["positions"], x["inv_freq"], x["qw"], x["kw"], v=x["v"] if with_v else None,
                            k_cache=joint[:, :, 0], v_cache=joint[:, :, 1] if with_v else None, rows=rows.to(cuda),
                            output_k=output_k)
    q2, k2 = gdn.qk_norm_rope(x["q"], x["k"], x["positions"], x["inv_freq"], x["qw"], x["kw"])
    torch.cuda.synchronize()
    assert torch.equal(q, q2) and (torch.equal(k, k2) if output_k else k is None)
    _hold(q2, k2, d, dtype)
    flat = before.view(-1, 2, Hk, D)
    at = (rows >= 0) & (rows < pages * size)
    flat[rows[at], 0] = k2.cpu()[at]
    if with_v:
        flat[rows[at], 1] = d["v"][at]
    assert torch.equal(joint.cpu(), before)


def test_not_finite_stays_where_it_is(gdn, cuda):
    """A head with an infinity or a NaN, a position's NaN frequency: the other heads, pairs and tokens are as without it."""
    announce("qk_norm_rope not finite")
    d = _inputs((50,), 8, 2, 64, 32, 11, F32)
    x = _to(d, cuda)
    clean, _ = gdn.qk_norm_rope(x["q"], x["k"], x["positions"], x["inv_freq"], x["qw"], x["kw"])
    x["q"][7, 3, 40] = float("nan")
    x["q"][9, 4, 60] = float("inf")  # (its norm is infinite: the head's other entries are 0 or NaN)
    q, _ = gdn.qk_norm_rope(x["q"], x["k"], x["positions"], x["inv_freq"], x["qw"], x["kw"])
    f = x["inv_freq"].clone()
    f[2] = float("nan")
    q3, _ = gdn.qk_norm_rope(_to(d, cuda)["q"], x["k"], x["positions"], f, x["qw"], x["kw"])
    torch.cuda.synchronize()
    same = torch.ones(50, 8, dtype=torch.bool)
    same[7, 3] = same[9, 4] = False
    assert torch.equal(q.cpu()[same], clean.cpu()[same]) and bool(q[7, 3].isnan().all())
    keep = [i for i in range(64) if i not in (2, 18)]
    assert torch.equal(q3[..., keep], clean[..., keep]) and bool(q3[..., [2, 18]].isnan().all())


def test_nothing_to_do(gdn, cuda):
    f = torch.ones(8, device=cuda)
    q, k = gdn.qk_norm_rope(torch.empty(0, 2, 64, device=cuda), torch.empty(0, 1, 64, device=cuda),
                            torch.empty(0, dtype=torch.long, device=cuda), f)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)


def test_cache_of_no_rows(gdn, cuda):
    """A cache without pages: no row is in it, and what comes back is what comes back without one."""
    announce("qk_norm_rope cache of no rows")
    g = torch.Generator().manual_seed(9)
    q, k, v = (A.randn(g, 5, h, 64, dtype=BF).to(cuda) for h in (4, 2, 2))
    at, f, none = torch.arange(5, device=cuda), torch.rand(32, generator=g).to(cuda), torch.empty(0, 16, 2, 64, dtype=BF, device=cuda)
    want = gdn.qk_norm_rope(q, k, at, f)
    for kw in (dict(v=v, v_cache=none.clone()), dict()):
        got = gdn.qk_norm_rope(q, k, at, f, k_cache=none, rows=at, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

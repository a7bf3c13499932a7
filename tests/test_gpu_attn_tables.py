"""Attention's tables with the forms that share keys out: packed sequences whose keys several workgroups share, infinities and NaN
inside packed sequences, pages outside the cache of streams that are cut into chunks (bounds: ``attn_testing``, values:
``attn_planted``)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import attn_planted as P
import attn_testing as A
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")
CODE = {F32: 0, BF: 1}
BEHIND = 3  # rows behind the last sequence

# queries and keys of each sequence, Hq, Hk, D, window, sinks; rows of a workgroup, whether several share their keys
PACKED = [([8, 8, 8, 8], [4104, 4104, 4104, 4104], 8, 2, 128, None, 0, BF, 32, True),
          ([5, 0, 9, 1, 30, 0], [5005, 700, 9, 3000, 12, 0], 8, 2, 128, None, 0, BF, 32, True),  # (fewer tiles than shares; more queries than keys)
          ([7, 3, 12], [2500, 3, 3500], 6, 2, 64, 1400, 40, BF, 32, True),
          ([3, 0, 20, 4], [2000, 5, 2600, 1], 4, 2, 64, None, 0, F32, 32, True),
          ([9, 2], [3000, 2100], 4, 2, 128, 1500, 5, F32, 32, True),
          ([60, 0, 1, 33, 90], [90, 40, 1, 233, 90], 4, 2, 64, 50, 3, BF, 128, False),
          ([700, 0, 650], [800, 40, 650], 4, 2, 64, None, 0, BF, 32, False),
          ([30, 70], [130, 70], 4, 2, 128, None, 0, F32, 32, False),
          ([1500, 0, 700, 3, 900], [1500, 9, 1100, 3, 850], 16, 4, 128, 200, 5, BF, 128, False),
          ([1500, 2400], [1600, 2400], 16, 8, 64, 150, 20, F32, 128, False)]


def _bounds(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32)


def _form(gdn, case):
    nq, nk, Hq, Hk, D, window, sinks, dtype = case[:8]
    form = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_fwd_form", 1, len(nq), sum(nq) + BEHIND, sum(nk) + BEHIND, Hq, Hk, D, window or 0,
                            sinks, CODE[dtype], form)
    return form[0], form[1] > 1


def _some(n):
    return torch.cat([torch.arange(min(3, n)), torch.arange(0, n, 101), torch.arange(max(0, n - 3), n)]).unique()


def _run(gdn, cuda, case, q, k, v):
    """A call on dirty memory: the rows behind the last sequence have to stay as they were."""
    nq, nk, Hq, Hk, D, window, sinks, dtype = case[:8]
    native = gdn.ops._native
    cu, cu_k = _bounds(nq).to(cuda), _bounds(nk).to(cuda)
    q, k, v = (torch.cat([x, torch.full((BEHIND, *x.shape[1:]), NAN, dtype=dtype)]).to(cuda) for x in (q, k, v))
    o = torch.full_like(q, 7.0)
    sizes = len(nq), len(q), len(k), Hq, Hk, D, window or 0, sinks
    need = native.lib().zattn_window_fwd_workspace_bytes(1, *sizes, CODE[dtype])
    w = torch.full((max(need, 1),), 0xFF, dtype=torch.uint8, device=cuda)
    native.call("zattn_window_fwd", q.data_ptr(), Hq * D, k.data_ptr(), Hk * D, v.data_ptr(), Hk * D, CODE[dtype], o.data_ptr(),
                cu.data_ptr(), cu_k.data_ptr(), len(nq), 1, len(q), len(k), Hq, Hk, D, window or 0, sinks, D**-0.5, w.data_ptr(),
                need, torch.cuda.current_stream().cuda_stream)
    again = gdn.window_attn_fwd(q[None], k[None], v[None], window=window, sinks=sinks, cu_seqlens=cu, cu_seqlens_k=cu_k)[0]
    o, again = o.cpu(), again.cpu()
    assert bool((o[-BEHIND:] == 7).all())
    o = o[:-BEHIND]
    assert torch.equal(o.isnan(), again[:-BEHIND].isnan()) and torch.equal(o.nan_to_num(0), again[:-BEHIND].nan_to_num(0))
    return o


@pytest.mark.parametrize("case", PACKED, ids=str)
def test_packed(gdn, cuda, case):
    nq, nk, Hq, Hk, D, window, sinks, dtype, rows, shared = case
    announce(f"window_attn_fwd packed {nq}/{nk} {Hq}/{Hk} D {D} window {window} sinks {sinks} {dtype}")
    assert _form(gdn, case) == (rows, shared)
    g = torch.Generator().manual_seed(81)
    q, k = P.queries_and_keys(g, (sum(nq),), (sum(nk),), Hq, Hk, D, dtype)
    v = torch.cat([P.planted(n, Hk, D, dtype)[0] for n in nk if n])
    o = _run(gdn, cuda, case, q, k, v)
    cu, cu_k = _bounds(nq).tolist(), _bounds(nk).tolist()
    for i, (n, m) in enumerate(zip(nq, nk)):
        if n:
            r, keys = _some(n), slice(cu_k[i], cu_k[i + 1])
            want = A.attend(q[cu[i] + r], k[keys], v[keys], m - n + r, window=window, sinks=sinks)
            e = A.within(o[cu[i] + r], want[0], A.attend_bound(*want, dtype, max(m, 1)))
            assert e <= 1, (i, e)


@pytest.mark.parametrize("case", PACKED, ids=str)
def test_packed_not_finite(gdn, cuda, case):
    """Infinities and NaN in some values of each sequence: rows that see none are to the bit as without, in other sequences too;
    entries where one is seen are not finite, the others of their rows to the bit as without."""
    nq, nk, Hq, Hk, D, window, sinks, dtype = case[:8]
    announce(f"window_attn_fwd packed not finite {nq}/{nk} {Hq}/{Hk} D {D} window {window} sinks {sinks} {dtype}")
    g = torch.Generator().manual_seed(82)
    q, k, v = (A.randn(g, sum(n), h, D, dtype=dtype) for n, h in ((nq, Hq), (nk, Hk), (nk, Hk)))
    cu, cu_k = _bounds(nq).tolist(), _bounds(nk).tolist()
    odd = torch.zeros(sum(nk), D, dtype=torch.bool)  # of key head Hk - 1
    for i, (n, m) in enumerate(zip(nq, nk)):
        places = {0, m - 1, m - n, m - n // 2, *torch.randint(0, max(m, 1), (2,), generator=g).tolist()}
        for t, j in enumerate(sorted(x for x in places if 0 <= x < m)):
            odd[cu_k[i] + j, (11 * i + 7 * t + 1) % D] = True
    v[:, Hk - 1][odd] = 0
    clean = _run(gdn, cuda, case, q, k, v)
    for t, (j, d) in enumerate(odd.nonzero().tolist()):
        v[j, Hk - 1, d] = (INF, NAN, -INF)[t % 3]
    o = _run(gdn, cuda, case, q, k, v)
    hit = torch.zeros(sum(nq), Hq, D, dtype=torch.bool)
    for i, (n, m) in enumerate(zip(nq, nk)):
        p, j = (m - n + torch.arange(n))[:, None], torch.arange(m)
        sees = (j <= p) & ((p - j < window) | (j < sinks) if window else True)
        hit[cu[i]: cu[i + 1], Hq - Hq // Hk:] = (sees.float() @ odd[cu_k[i]: cu_k[i + 1]].float() > 0)[:, None]
    assert bool(hit.any()) and not bool(torch.isfinite(o[hit].float()).any())
    assert torch.equal(o[~hit], clean[~hit])


# lengths, room, page size, Hq, Hk, D, window, sinks: several chunks a stream
CUT = [([9000, 8999, 70], 9216, 64, 8, 2, 128, None, 0, BF), ([6000, 5000], 6144, 16, 4, 2, 64, 4500, 70, F32),
       ([20000], 20032, 64, 4, 1, 128, None, 0, F32), ([5000, 4097, 2048, 1], 5120, 512, 17, 1, 64, 3000, 600, BF)]


@pytest.mark.parametrize("case", CUT, ids=str)
@pytest.mark.parametrize("gone", ["some", "runs", "all but one", "all"])
def test_pages_outside_the_cache_of_cut_streams(gdn, cuda, case, gone):
    """Single pages, runs of pages as long as a chunk and longer, all but one and all: what is left is as if alone there."""
    lengths, room, page, Hq, Hk, D, window, sinks, dtype = case
    announce(f"window_attn_step without pages: {gone}, {case}")
    B, each = len(lengths), room // page
    form = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_step_form", B, room, Hq, Hk, window or 0, sinks, CODE[dtype], form)
    assert form[0] == 0 and form[1] > 1
    g = torch.Generator().manual_seed(83)
    q, k = P.queries_and_keys(g, (B,), (B, room), Hq, Hk, D, dtype)
    v = torch.stack([P.planted(room, Hk, D, dtype)[0]] * B)
    pages = torch.randperm(B * each, generator=g).view(B, each)
    kc, vc = (torch.empty(B * each, page, Hk, D, dtype=dtype) for _ in range(2))
    kc[pages.flatten()], vc[pages.flatten()] = k.view(-1, page, Hk, D), v.view(-1, page, Hk, D)
    there = torch.ones(B, each, dtype=torch.bool)
    for b, n in enumerate(lengths):
        last = (n - 1) // page
        if gone == "some":
            there[b, torch.randperm(each, generator=g)[: max(1, each // 5)]] = False
        elif gone == "runs":  # the first third of the pages and the last sixth
            there[b, : last // 3 + 1] = False
            there[b, last - last // 6:] = False
        else:
            there[b] = False
            if gone == "all but one":
                there[b, last // 2 if window is None else max(0, last - 1)] = True
    outside = torch.tensor([-1, B * each, 1 << 30, -(1 << 31)])[torch.arange(B * each).view(B, each) % 4]
    table = torch.where(there, pages, outside).int()
    for b in range(B):  # (and whatever lies on pages that no table names)
        kc[pages[b][~there[b]]] = vc[pages[b][~there[b]]] = NAN
    o = gdn.window_attn_step(q.to(cuda), kc.to(cuda), vc.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
                             window=window, sinks=sinks, pages=table.to(cuda)).cpu()
    j = torch.arange(room)
    for b, n in enumerate(lengths):
        sees = (j < n) & there[b, j // page]
        if window is not None:
            sees &= (n - 1 - j < window) | (j < sinks)
        m = int(sees.sum())
        if m == 0:
            assert not bool(o[b].any())
            continue
        want = A.attend(q[b: b + 1], k[b, sees], v[b, sees], torch.tensor([m - 1]))
        e = A.within(o[b: b + 1], want[0], A.attend_bound(*want, dtype, n))
        assert e <= 1, (b, m, e)

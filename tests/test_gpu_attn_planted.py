"""Attention over values that show single keys (``attn_planted``): a key, tile or chunk that is lost, taken twice, read for another
or seen from outside a window is off by more than the bound, in every form. The oracle is shown to hold that on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import attn_planted as P
import attn_testing as A
from gdn_testing import announce

BF, F32 = torch.bfloat16, torch.float32
CODE = {F32: 0, BF: 1}

# lengths of the streams, room, page size (None: a dense cache), Hq, Hk, D, window, sinks; one launch of wide workgroups, several
# chunks a stream
STEPS = [([20000], 20032, 64, 4, 2, 128, None, 0, BF, False, True), ([20000], 20032, 64, 4, 2, 128, None, 0, F32, False, True),
         ([6000, 5999, 1, 2049], 6016, 16, 8, 2, 128, None, 0, BF, False, True),
         ([4999, 33, 3000], 5000, None, 4, 2, 64, 3000, 37, F32, False, True),
         ([4097, 4096, 4095, 0], 4352, 256, 17, 1, 64, 2100, 100, BF, False, True),
         ([1024, 1000, 17], 1024, 64, 8, 2, 128, None, 0, BF, True, False),
         ([700, 699], 700, None, 5, 1, 64, 90, 40, F32, True, False),
         ([129 - n % 3 for n in range(300)], 130, None, 4, 2, 64, None, 0, BF, False, False)]
# Tq, Tk, Hq, Hk, D, window, sinks; rows of a workgroup, whether several share their keys
PROMPTS = [(5000, 5000, 8, 2, 128, None, 0, BF, 128, False), (2100, 2100, 16, 8, 128, 300, 37, BF, 128, False),
           (4200, 4200, 20, 4, 64, 500, 130, BF, 128, False), (3500, 3500, 12, 6, 64, 300, 1, F32, 128, False),
           (3000, 3000, 8, 4, 128, 200, 7, F32, 128, False),
           (600, 600, 8, 2, 128, None, 0, BF, 32, False), (900, 900, 5, 1, 64, 800, 9, BF, 32, False),
           (500, 500, 4, 2, 128, 300, 2, F32, 32, False), (500, 500, 4, 2, 64, None, 0, F32, 32, False),
           (20, 6000, 8, 2, 128, None, 0, BF, 32, True), (33, 5000, 6, 2, 64, 3000, 70, BF, 32, True),
           (9, 4000, 4, 2, 128, None, 0, F32, 32, True), (17, 2500, 4, 2, 64, 1500, 40, F32, 32, True)]


def _edges(p, window, sinks):
    """Keys at the ends of what the query at position p sees, inside and outside."""
    ends = [p, p + 1]
    if window is not None:
        ends += [p - window, p - window + 1, sinks - 1, sinks]
    return ends


def _step(case):
    """Of each stream: (q [Hq, D], k, v [n, Hk, D], planted keys, their columns)."""
    lengths, _, _, Hq, Hk, D, window, sinks, dtype = case[:9]
    g = torch.Generator().manual_seed(71)
    out = []
    for n in lengths:
        q, k = P.queries_and_keys(g, (), (n,), Hq, Hk, D, dtype)
        out.append((q, k, *(P.planted(n, Hk, D, dtype, _edges(n - 1, window, sinks)) if n else (k, None, None))))
    return out


def _prompt(case):
    Tq, Tk, Hq, Hk, D, window, sinks, dtype = case[:8]
    g = torch.Generator().manual_seed(72)
    q, k = P.queries_and_keys(g, (Tq,), (Tk,), Hq, Hk, D, dtype)
    rows = torch.cat([torch.arange(min(3, Tq)), torch.randperm(Tq, generator=g)[:8], torch.arange(max(0, Tq - 3), Tq)]).unique()
    ends = [e for r in rows.tolist() for e in _edges(Tk - Tq + r, window, sinks)]
    return q, k, *P.planted(Tk, Hk, D, dtype, ends), rows


@pytest.mark.parametrize("case", STEPS, ids=str)
def test_mistakes_show_in_steps(case):
    window, sinks, dtype = case[6:9]
    for n, (q, k, v, keys, columns) in list(zip(case[0], _step(case)))[:4]:
        if n > 1:
            assert P.least_mistake(q, k, v, keys, columns, n - 1, window, sinks, dtype) > 1.5


@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_mistakes_show_in_prompts(case):
    Tq, Tk, window, sinks, dtype = case[0], case[1], *case[5:8]
    q, k, v, keys, columns, rows = _prompt(case)
    for r in rows.tolist():
        if Tk - Tq + r > 0:
            assert P.least_mistake(q[r], k, v, keys, columns, Tk - Tq + r, window, sinks, dtype) > 1.5


@pytest.mark.gpu
@pytest.mark.parametrize("case", STEPS, ids=str)
def test_steps(gdn, cuda, case):
    lengths, room, page, Hq, Hk, D, window, sinks, dtype, wide, shared = case
    announce(f"window_attn_step planted {lengths[:4]} of {room} page {page} {Hq}/{Hk} D {D} window {window} sinks {sinks} {dtype}")
    B = len(lengths)
    form = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_step_form", B, room, Hq, Hk, window or 0, sinks, CODE[dtype], form)
    assert (bool(form[0]), form[1] > 1) == (wide, shared)
    streams = _step(case)
    size = page or room
    each = room // size
    pages = torch.randperm(B * each, generator=torch.Generator().manual_seed(73)).view(B, each)
    if page is None:
        pages = torch.arange(B)[:, None]
    kc, vc = (torch.full((B * each, size, Hk, D), float("nan"), dtype=dtype) for _ in range(2))
    for b, (_, k, v, _, _) in enumerate(streams):
        p = torch.arange(k.shape[0])
        row = pages[b, p // size] * size + p % size
        kc.view(-1, Hk, D)[row], vc.view(-1, Hk, D)[row] = k, v
    q = torch.stack([s[0] for s in streams])
    o = gdn.window_attn_step(q.to(cuda), kc.to(cuda), vc.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
                             window=window, sinks=sinks, pages=None if page is None else pages.int().to(cuda)).cpu()
    for b, n in enumerate(lengths):
        want = A.attend(q[b: b + 1], streams[b][1], streams[b][2], torch.tensor([n - 1]), window=window, sinks=sinks)
        e = A.within(o[b: b + 1], want[0], A.attend_bound(*want, dtype, n))
        assert e <= 1, (b, n, e)


@pytest.mark.gpu
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_prompts(gdn, cuda, case):
    Tq, Tk, Hq, Hk, D, window, sinks, dtype, tile_rows, shared = case
    announce(f"window_attn_fwd planted {Tq}/{Tk} {Hq}/{Hk} D {D} window {window} sinks {sinks} {dtype}")
    form = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_fwd_form", 0, 1, Tq, Tk, Hq, Hk, D, window or 0, sinks, CODE[dtype], form)
    assert (form[0], form[1] > 1) == (tile_rows, shared)
    q, k, v, _, _, rows = _prompt(case)
    o = gdn.window_attn_fwd(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), window=window, sinks=sinks)[0].cpu()
    want = A.attend(q[rows], k, v, Tk - Tq + rows, window=window, sinks=sinks)
    e = A.within(o[rows], want[0], A.attend_bound(*want, dtype, Tk))
    assert e <= 1, e

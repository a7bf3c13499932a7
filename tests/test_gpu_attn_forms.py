"""The attention kernels in each of their forms, by sizes that are asserted to take it: values that are not finite, repeats over
dirty memory, graphs, streams, guarded buffers, offsets past 32 bits (bounds: ``attn_testing``)."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

import attn_testing as A
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")
CODE = {F32: 0, BF: 1}


def _fwd_form(gdn, B, Tq, Tk, Hq, Hk, D, window, sinks, dtype, packed=0):
    out = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_fwd_form", packed, B, Tq, Tk, Hq, Hk, D, window or 0, sinks, CODE[dtype], out)
    return out[0], out[1] > 1


def _step_form(gdn, B, room, Hq, Hk, window, sinks, dtype):
    out = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_step_form", B, room, Hq, Hk, window or 0, sinks, CODE[dtype], out)
    return bool(out[0]), out[1] > 1


# (B, Tq, Tk, Hq, Hk, D, window, sinks, dtype), rows of a workgroup, whether several share their keys
FORMS = [((1, 2100, 2100, 16, 8, 128, 300, 5, BF), 128, False), ((3, 1400, 1400, 20, 4, 64, 200, 130, BF), 128, False),
         ((1, 3000, 3000, 8, 4, 128, 200, 7, F32), 128, False), ((1, 3500, 3500, 12, 6, 64, 300, 1, F32), 128, False),
         ((1, 600, 600, 8, 2, 128, None, 0, BF), 32, False), ((1, 900, 900, 5, 1, 64, 800, 9, BF), 32, False),
         ((1, 500, 500, 4, 2, 128, 300, 2, F32), 32, False), ((1, 500, 500, 4, 2, 64, None, 0, F32), 32, False),
         ((1, 20, 3000, 8, 2, 128, None, 0, BF), 32, True), ((1, 33, 2500, 6, 2, 64, 2000, 3, BF), 32, True),
         ((1, 9, 2500, 4, 2, 128, None, 0, F32), 32, True), ((2, 17, 2500, 4, 2, 64, 1500, 40, F32), 32, True)]


def _inputs(B, Tq, Tk, Hq, Hk, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [A.randn(g, B, Tq, Hq, D, dtype=dtype), A.randn(g, B, Tk, Hk, D, dtype=dtype), A.randn(g, B, Tk, Hk, D, dtype=dtype)]


def _some(T, n=12):
    return torch.cat([torch.arange(min(3, T)), torch.randperm(T, generator=torch.Generator().manual_seed(2))[:n],
                      torch.arange(max(0, T - 3), T)]).unique()


def _hold(o, q, k, v, rows, dtype, **kw):
    want = A.attend(q[rows], k, v, k.shape[0] - q.shape[0] + rows, **kw)
    e = A.within(o.cpu()[rows], want[0], A.attend_bound(*want, dtype, k.shape[0]))
    assert e <= 1, e


@pytest.mark.parametrize("sizes,rows,shared", FORMS)
def test_forms(gdn, cuda, sizes, rows, shared):
    """Each form against float64, on queries and keys that are slices of one projection's rows."""
    B, Tq, Tk, Hq, Hk, D, window, sinks, dtype = sizes
    announce(f"window_attn_fwd form {rows} {shared}: {sizes}")
    assert _fwd_form(gdn, *sizes) == (rows, shared)
    q, k, v = _inputs(B, Tq, Tk, Hq, Hk, D, dtype, 41)
    kv = torch.cat([k.flatten(2), v.flatten(2)], -1).to(cuda)
    x, y = (t.unflatten(-1, (Hk, D)) for t in kv.split(Hk * D, -1))
    o = gdn.window_attn_fwd(q.to(cuda), x, y, window=window, sinks=sinks)
    torch.cuda.synchronize()
    for b in range(B):
        _hold(o[b], q[b], k[b], v[b], _some(Tq), dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("sizes,rows,shared", FORMS)
def test_not_finite(gdn, cuda, sizes, rows, shared):
    """Infinities and NaN in values, all over a few keys: rows that see none of them are to the bit as without them, and so is
    every entry that none of those that its row sees stands at; entries where one does are not finite."""
    B, Tq, Tk, Hq, Hk, D, window, sinks, dtype = sizes
    announce(f"window_attn_fwd not finite, form {rows} {shared}: {sizes}")
    q, k, v = _inputs(B, Tq, Tk, Hq, Hk, D, dtype, 42)
    kw = dict(window=window, sinks=sinks)
    keys = torch.randperm(Tk, generator=torch.Generator().manual_seed(3))[:4].tolist() + [Tk - 1, max(0, Tk - Tq), 0]
    odd = torch.zeros(Tk, D, dtype=torch.bool)
    for n, j in enumerate(keys):
        odd[j, (7 * n + 1) % D] = True
    zeroed = v.clone()
    zeroed[0, :, 0][odd] = 0
    clean = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), zeroed.to(cuda), **kw).cpu()
    for n, (j, d) in enumerate(odd.nonzero().tolist()):
        v[0, j, 0, d] = (INF, NAN, -INF)[n % 3]
    o = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), **kw).cpu()
    torch.cuda.synchronize()
    p, j = (Tk - Tq + torch.arange(Tq))[:, None], torch.arange(Tk)
    sees = (j <= p) & ((p - j < window) | (j < sinks) if window else True)
    hit = (sees.float() @ odd.float() > 0)[:, None].expand(Tq, Hq, D).clone()  # [Tq, Hq, D]
    hit[:, Hq // Hk:] = False
    assert not bool(torch.isfinite(o[0][hit].float()).any())
    assert torch.equal(o[0][~hit], clean[0][~hit]) and torch.equal(o[1:], clean[1:])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_windows_and_sinks_that_hold_all(gdn, cuda, dtype):
    """A window of all keys or of more, and sinks of all, are no window: to the bit, dense, packed and for one token."""
    announce(f"windows of all keys {dtype}")
    q, k, v = (t.to(cuda) for t in _inputs(1, 150, 190, 4, 2, 64, dtype, 44))
    n = torch.tensor([190], dtype=torch.int32, device=cuda)
    for call in (lambda **kw: gdn.window_attn_fwd(q, k, v, **kw), lambda **kw: gdn.window_attn_step(q[:, -1], k, v, n, **kw),
                 lambda **kw: gdn.window_attn_fwd(q, k, v, cu_seqlens=[0, 40, 150], cu_seqlens_k=[0, 60, 190], **kw)):
        plain = call()
        for kw in (dict(window=190), dict(window=191, sinks=3), dict(window=1 << 31), dict(window=1 << 40, sinks=1 << 40)):
            assert torch.equal(call(**kw), plain), kw
    o = gdn.window_attn_fwd(q, k, v, window=5, sinks=1 << 40)
    _hold(o[0], q[0].cpu(), k[0].cpu(), v[0].cpu(), torch.arange(150), dtype, window=5, sinks=190)


@pytest.mark.parametrize("sizes,rows,shared", FORMS[::2])
def test_repeats_over_dirty_memory(gdn, cuda, sizes, rows, shared):
    """The same to the bit, whatever a call's LDS and workspace held: between them calls whose values are all NaN."""
    B, Tq, Tk, Hq, Hk, D, window, sinks, dtype = sizes
    announce(f"window_attn_fwd repeats, form {rows} {shared}: {sizes}")
    q, k, v = (t.to(cuda) for t in _inputs(B, Tq, Tk, Hq, Hk, D, dtype, 43))
    first = gdn.window_attn_fwd(q, k, v, window=window, sinks=sinks)
    for _ in range(3):
        bad = gdn.window_attn_fwd(q, k, torch.full_like(v, NAN), window=window, sinks=sinks)
        again = gdn.window_attn_fwd(q, k, v, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert torch.equal(first, again) and not bool(torch.isfinite(bad.float()).any())


STEPS = [((1, 900, 8, 2, 128, None, 0, BF), True, False), ((3, 400, 6, 3, 64, 100, 2, F32), True, False),
         ((2, 6000, 8, 2, 128, None, 0, BF), False, True), ((1, 5000, 4, 2, 64, 3000, 4, F32), False, True),
         ((300, 130, 4, 2, 64, None, 0, BF), False, False), ((300, 200, 2, 2, 128, 60, 3, F32), False, False)]


def _step_inputs(B, room, Hq, Hk, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(1, room + 1, (B,), generator=g)
    return [A.randn(g, B, Hq, D, dtype=dtype), A.randn(g, B, room, Hk, D, dtype=dtype), A.randn(g, B, room, Hk, D, dtype=dtype),
            lengths.int()]


@pytest.mark.parametrize("sizes,wide,shared", STEPS)
def test_step_forms(gdn, cuda, sizes, wide, shared):
    B, room, Hq, Hk, D, window, sinks, dtype = sizes
    announce(f"window_attn_step form {wide} {shared}: {sizes}")
    assert _step_form(gdn, B, room, Hq, Hk, window, sinks, dtype) == (wide, shared)
    q, kc, vc, lengths = _step_inputs(B, room, Hq, Hk, D, dtype, 44)
    x = [t.to(cuda) for t in (q, kc, vc, lengths)]
    o = gdn.window_attn_step(*x, window=window, sinks=sinks)
    bad = [t.clone() for t in x]
    for t in bad[1:3]:  # what is not seen has no part, to the bit
        for b, n in enumerate(lengths.tolist()):
            t[b, n:] = NAN
            if window:
                t[b, min(sinks, max(0, n - window)): max(0, n - window)] = INF
    o2 = gdn.window_attn_step(*bad, window=window, sinks=sinks)
    o3 = gdn.window_attn_step(*x, window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert torch.equal(o, o2) and torch.equal(o, o3)
    for b in range(0, B, max(1, B // 6)):
        n = int(lengths[b])
        _hold(o[b: b + 1], q[b: b + 1], kc[b, :n], vc[b, :n], torch.tensor([0]), dtype, window=window, sinks=sinks)


def _sublayer(gdn, s):
    q, k = gdn.qk_norm_rope(s["q"], s["k"], s["at"], s["freq"], v=s["v"], k_cache=s["kc"], v_cache=s["vc"], rows=s["rows"])
    return (gdn.window_attn_fwd(q, k, s["v"], window=70, sinks=3),
            gdn.window_attn_fwd(q[:, -5:], k, s["v"], sinks=3),
            gdn.window_attn_step(q[0, -3:], s["kc"], s["vc"], s["lengths"], pages=s["pages"]))


def _sublayer_inputs(cuda, seed, T=900):
    g = torch.Generator().manual_seed(seed)
    r = lambda *z: A.randn(g, *z, dtype=BF).to(cuda)  # noqa: E731
    return {"q": r(1, T, 8, 128), "k": r(1, T, 2, 128), "v": r(1, T, 2, 128), "kc": torch.zeros(1024, 16, 2, 128, dtype=BF, device=cuda),
            "vc": torch.zeros(1024, 16, 2, 128, dtype=BF, device=cuda), "at": torch.arange(T, device=cuda)[None],
            "freq": torch.rand(64, generator=g).to(cuda), "rows": (torch.randperm(1024 * 16, generator=g)[:T]).to(cuda)[None],
            "pages": torch.randint(0, 1024, (3, 300), generator=g).int().to(cuda),
            "lengths": torch.tensor([4800, 1, 333], dtype=torch.int32, device=cuda)}


def test_graphs_and_streams(gdn, cuda):
    """Two captured graphs, replayed in turn and beside eager calls on a stream of their own, each with its own results."""
    announce("attention sublayer in two graphs, replays between eager calls")
    a, b = _sublayer_inputs(cuda, 51), _sublayer_inputs(cuda, 52)
    eager = [_sublayer(gdn, a), _sublayer(gdn, b)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for s in (a, b):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _sublayer(gdn, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_sublayer(gdn, s))
        graphs.append(g)
    for n in range(3):
        for o in outs:
            for t in o:
                t.fill_(NAN)
        graphs[n % 2].replay()
        with torch.cuda.stream(side):
            beside = _sublayer(gdn, _sublayer_inputs(cuda, 53))
        graphs[1 - n % 2].replay()
        torch.cuda.synchronize()
        again = _sublayer(gdn, a)
        torch.cuda.synchronize()
        for got, want in ((outs[0], eager[0]), (outs[1], eager[1]), (again, eager[0])):
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        del beside


def test_guarded_buffers(gdn, cuda):
    """Outputs and workspaces of just the size that a call needs, between guard regions, through the C ABI."""
    announce("zattn_window_fwd, zattn_window_step between guards")
    native = gdn.ops._native
    stream = torch.cuda.current_stream().cuda_stream

    def guarded(nbytes):
        t = torch.full((nbytes + 4096,), 0x5A, dtype=torch.uint8, device=cuda)
        return t, t[2048: 2048 + nbytes], t[2048:].data_ptr()

    def check(t, nbytes):
        assert bool((t[:2048] == 0x5A).all()) and bool((t[2048 + nbytes:] == 0x5A).all())

    for sizes in (FORMS[0][0], FORMS[4][0], FORMS[8][0], FORMS[11][0]):
        B, Tq, Tk, Hq, Hk, D, window, sinks, dtype = sizes
        q, k, v = (t.to(cuda) for t in _inputs(B, Tq, Tk, Hq, Hk, D, dtype, 45))
        need = native.lib().zattn_window_fwd_workspace_bytes(0, B, Tq, Tk, Hq, Hk, D, window or 0, sinks, CODE[dtype])
        n = q.numel() * q.element_size()
        (o, inner, at), (w, _, wat) = guarded(n), guarded(need)
        native.call("zattn_window_fwd", q.data_ptr(), Hq * D, k.data_ptr(), Hk * D, v.data_ptr(), Hk * D, CODE[dtype], at, None,
                    None, 0, B, Tq, Tk, Hq, Hk, D, window or 0, sinks, D**-0.5, wat, need, stream)
        torch.cuda.synchronize()
        check(o, n)
        check(w, need)
        want = gdn.window_attn_fwd(q, k, v, window=window, sinks=sinks)
        assert torch.equal(inner.view(dtype).view(q.shape), want)
    for sizes, _, _ in STEPS[::2]:
        B, room, Hq, Hk, D, window, sinks, dtype = sizes
        q, kc, vc, lengths = (t.to(cuda) for t in _step_inputs(B, room, Hq, Hk, D, dtype, 46))
        need = native.lib().zattn_window_step_workspace_bytes(B, room, Hq, Hk, D, window or 0, sinks, CODE[dtype])
        n = q.numel() * q.element_size()
        (o, inner, at), (w, _, wat) = guarded(n), guarded(need)
        native.call("zattn_window_step", q.data_ptr(), Hq * D, kc.data_ptr(), Hk * D, vc.data_ptr(), Hk * D, CODE[dtype],
                    lengths.data_ptr(), None, room, 1, B * room, at, B, Hq, Hk, D, window or 0, sinks, D**-0.5, wat, need, stream)
        torch.cuda.synchronize()
        check(o, n)
        check(w, need)
        assert torch.equal(inner.view(dtype).view(q.shape), gdn.window_attn_step(q, kc, vc, lengths, window=window, sinks=sinks))


def test_packed_rows_behind_the_last_sequence(gdn, cuda):
    """Packed forms write their sequences' rows and no others."""
    announce("zattn_window_fwd packed, rows of no sequence")
    native = gdn.ops._native
    for Tq, Hq, D, window, rows in ((2600, 16, 128, 100, 128), (1000, 4, 64, 0, 32)):
        q, k, v = (t.to(cuda) for t in _inputs(1, Tq, Tq, Hq, 2, D, BF, 47))
        assert _fwd_form(gdn, 5, Tq, Tq, Hq, 2, D, window, 0, BF, packed=1)[0] == rows
        ends = [0, 3, 3, Tq // 3, Tq // 2, Tq - 70]
        cu = torch.tensor(ends, dtype=torch.int32, device=cuda)
        o = torch.full_like(q, 7.0)
        need = native.lib().zattn_window_fwd_workspace_bytes(1, 5, Tq, Tq, Hq, 2, D, window, 0, 1)
        w = torch.empty(max(need, 1), dtype=torch.uint8, device=cuda)
        native.call("zattn_window_fwd", q.data_ptr(), Hq * D, k.data_ptr(), 2 * D, v.data_ptr(), 2 * D, 1, o.data_ptr(), cu.data_ptr(),
                    cu.data_ptr(), 5, 1, Tq, Tq, Hq, 2, D, window, 0, D**-0.5, w.data_ptr(), need,
                    torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert bool((o[:, Tq - 70:] == 7).all())
        for a, b in zip(ends, ends[1:]):
            if b > a:
                _hold(o[0, a:b], q[0, a:b].cpu(), k[0, a:b].cpu(), v[0, a:b].cpu(), _some(b - a, 4), BF, window=window or None)


def test_offsets_past_32_bits(gdn, cuda):
    """Rows of keys 4 MiB apart over more than 4 GiB, caches whose pages lie behind 4 GiB."""
    announce("attention over rows behind 4 GiB")
    T, D, Hk = 1200, 64, 2
    g = torch.Generator().manual_seed(48)
    wide = torch.empty(T, 1 << 21, dtype=BF, device=cuda)  # 4 MiB a row, 5 GiB
    q = A.randn(g, 1, T, 4, D, dtype=BF)
    k, v = A.randn(g, T, Hk, D, dtype=BF), A.randn(g, T, Hk, D, dtype=BF)
    x, y = (wide[:, at: at + Hk * D].unflatten(-1, (Hk, D)) for at in (0, 4096))
    x.copy_(k)
    y.copy_(v)
    for kw in ({}, {"window": 100, "sinks": 4}):
        o = gdn.window_attn_fwd(q.to(cuda), x[None], y[None], **kw)
        o2 = gdn.window_attn_fwd(q[:, -4:].to(cuda), x[None], y[None], **kw)
        torch.cuda.synchronize()
        _hold(o[0], q[0], k, v, _some(T, 6), BF, **kw)
        _hold(o2[0], q[0, -4:], k, v, torch.arange(4), BF, **kw)
    cache = wide.view(-1, 64, Hk, D)  # pages of 16 KiB, 327680 of them
    n, last = 700, cache.shape[0]
    pages = torch.stack([last - 1 - torch.arange(11), torch.arange(11) * 29000 + 3])
    rows = (pages[:, torch.arange(n) // 64] * 64 + torch.arange(n) % 64).to(cuda)
    qs, ks, vs = A.randn(g, 2, n, 4, D, dtype=BF), A.randn(g, 2, n, Hk, D, dtype=BF), A.randn(g, 2, n, Hk, D, dtype=BF)
    vc = torch.empty_like(cache)
    freq = torch.zeros(8, device=cuda)  # (nothing turns: the cache holds the norms)
    qn, kn = gdn.qk_norm_rope(qs.to(cuda), ks.to(cuda), torch.zeros(2, n, dtype=torch.long, device=cuda), freq, v=vs.to(cuda),
                              k_cache=cache, v_cache=vc, rows=rows)
    assert torch.equal(cache.view(-1, Hk, D)[rows], kn) and torch.equal(vc.view(-1, Hk, D)[rows], vs.to(cuda))
    o = gdn.window_attn_step(qn[:, -1].contiguous(), cache, vc, torch.full((2,), n, dtype=torch.int32, device=cuda),
                             pages=pages.int().to(cuda))
    torch.cuda.synchronize()
    for b in range(2):
        _hold(o[b: b + 1], qn[b, -1:].cpu(), kn[b].cpu(), vs[b], torch.tensor([0]), BF)


def test_copies_and_empty_calls(gdn, cuda):
    """Layouts that no kernel reads in place (heads ahead of tokens, rows at odd addresses) are copied; calls of nothing."""
    announce("attention on transposed and unaligned tensors, empty calls")
    q, k, v = _inputs(1, 50, 50, 4, 2, 64, BF, 49)
    want = gdn.window_attn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), window=9)
    t = [x.transpose(1, 2).contiguous().to(cuda).transpose(1, 2) for x in (q, k, v)]
    odd = [torch.cat([x.flatten().new_zeros(3), x.flatten()]).to(cuda)[3:].view(x.shape) for x in (q, k, v)]
    assert torch.equal(gdn.window_attn_fwd(*t, window=9), want) and torch.equal(gdn.window_attn_fwd(*odd, window=9), want)
    at, f = torch.arange(50, device=cuda)[None], torch.rand(16, device=cuda)
    a, b = gdn.qk_norm_rope(q.to(cuda), k.to(cuda), at, f), gdn.qk_norm_rope(t[0], odd[1], at, f)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert gdn.window_attn_fwd(t[0][:, :0], t[1], t[2]).shape == (1, 0, 4, 64)
    assert not bool(gdn.window_attn_fwd(q.to(cuda), t[1][:, :0], t[2][:, :0]).any())
    n = torch.zeros(3, dtype=torch.int32, device=cuda)
    q3, c = torch.ones(3, 4, 64, device=cuda), torch.ones(3, 0, 2, 64, device=cuda)
    assert not bool(gdn.window_attn_step(q3, c, c, n).any())
    c = torch.ones(2, 16, 2, 64, device=cuda)
    assert not bool(gdn.window_attn_step(q3, c, c, n + 5, pages=torch.zeros(3, 0, dtype=torch.int32, device=cuda)).any())
    assert gdn.window_attn_step(q3[:0], c, c, n[:0], pages=torch.zeros(0, 4, dtype=torch.int32, device=cuda)).shape == (0, 4, 64)
    torch.cuda.synchronize()


def test_threads_on_streams_of_their_own(gdn, cuda):
    """Four threads, a stream and a window each, at one time: each its own results, of both forms and the step."""
    announce("attention sublayer from four threads")
    q, k, v = (t.to(cuda) for t in _inputs(1, 700, 700, 8, 2, 128, BF, 45))
    n = torch.tensor([700], dtype=torch.int32, device=cuda)
    calls = lambda i: (gdn.window_attn_fwd(q, k, v, window=100 + i, sinks=i),  # noqa: E731
                       gdn.window_attn_fwd(q[:, -20:], k, v), gdn.window_attn_step(q[:, -1], k, v, n, window=300 + i))
    want, got = [calls(i) for i in range(4)], [None] * 4
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = calls(i)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))

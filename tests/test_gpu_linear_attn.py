"""Linear attention with a decay per head (``ops.linear_attn_fwd``, ``ops.linear_attn_step``) against the token-by-token
recurrence in float64: lengths around segments and stages, head layouts, types, packed and empty sequences, strides,
resets, states in place, non-finite values, graphs and streams. Bounds: ``linear_testing``."""

from __future__ import annotations

import math

import pytest
import torch

import linear_testing as L
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _check(gdn, cuda, d, cu=None, g=None, scale=None, msg="", **kw):
    g = d["g"] if g is None else g
    s0 = d["s0"]
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=cuda)
    o, s = gdn.ops.linear_attn_fwd(*(t.to(cuda) for t in (d["q"], d["k"], d["v"], g)), scale=scale,
                                   initial_state=None if s0 is None else s0.to(cuda), cu_seqlens=cut, **kw)
    torch.cuda.synchronize()
    o_ref, s_ref, o_mag, s_mag = L.tokens(d["q"], d["k"], d["v"], g, s0, scale, cu)
    T, K = d["q"].shape[1], d["q"].shape[3]
    eo = L.within(o, o_ref, L.out_bound(o_ref, o_mag, d["q"].dtype, T, K))
    es = L.within(s, s_ref, L.state_bound(s_mag, T))
    print(f"[errors] {msg} outputs {eo:.3f}, states {es:.3f} of their bounds")
    assert o.dtype == d["q"].dtype and s.dtype == F32 and eo <= 1 and es <= 1, (eo, es)
    return o, s


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(gdn, cuda, T, dtype):
    announce(f"linear attn T={T} {dtype}")
    _check(gdn, cuda, L.inputs((2, T), 2, 2, 128, 128, T, dtype, n_states=2), msg=f"T={T} {dtype}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hk,Hv,K,V", [(1, 1, 64, 64), (1, 4, 128, 64), (2, 6, 64, 128), (3, 3, 128, 128), (1, 16, 128, 64)])
def test_head_layouts(gdn, cuda, Hk, Hv, K, V, dtype):
    announce(f"linear attn Hk={Hk} Hv={Hv} K={K} V={V} {dtype}")
    _check(gdn, cuda, L.inputs((1, 197), Hk, Hv, K, V, 7 * Hv + K, dtype), scale=0.3, msg=f"{Hk}/{Hv} {K}x{V}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[0], [0, 1, 0, 64, 65, 0], [128, 129, 3, 200, 1, 1, 1], [1] * 70 + [130] + [0] * 5 + [2]])
def test_packed(gdn, cuda, lengths, dtype):
    announce(f"linear attn packed {lengths[:8]} {dtype}")
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    d = L.inputs((1, cu[-1]), 1, 2, 64 if dtype == F32 else 128, 64, len(lengths), dtype, n_states=len(lengths))
    _check(gdn, cuda, d, cu, msg=f"packed {lengths[:8]}")


@pytest.mark.parametrize("dtype,T,H", [(BF, 2500, 1), (BF, 1500, 3), (F32, 1100, 1), (BF, 700, 16)])
def test_several_runs(gdn, cuda, dtype, T, H):
    """Sequences long enough to be summed as several runs whose states are carried on, with slow decays, so that most of
    a state is old."""
    announce(f"linear attn runs T={T} H={H} {dtype}")
    _check(gdn, cuda, L.inputs((1, T), H, H, 128, 128, T + H, dtype, n_states=1, slow=0.02), msg=f"runs T={T}")


def test_packed_runs(gdn, cuda):
    """Packed sequences of one and of several runs beside one another."""
    announce("linear attn packed runs")
    lengths = [1400, 0, 77, 900, 512]
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    _check(gdn, cuda, L.inputs((1, cu[-1]), 1, 1, 128, 128, 3, BF, n_states=5, slow=0.1), cu)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decay_forms(gdn, cuda, dtype):
    """A decay a head, bf16 decays, no decay, decays that leave fp32's range within a few tokens, resets."""
    announce(f"linear attn decays {dtype}")
    d = L.inputs((2, 150), 2, 4, 64, 64, 11, dtype, n_states=2)
    _check(gdn, cuda, d, g=torch.tensor([-0.5, -0.01, 0.0, -1e-5]), msg="fixed")
    _check(gdn, cuda, d, g=d["g"].to(BF), msg="bf16")
    _check(gdn, cuda, d, g=torch.zeros(2, 150, 4), msg="none")
    _check(gdn, cuda, d, g=d["g"] * 100, msg="strong")
    r = L.inputs((2, 333), 2, 2, 128, 64, 12, dtype, n_states=2, resets=0.02)
    assert bool(torch.isinf(r["g"]).any())
    o, s = _check(gdn, cuda, r, msg="resets")
    lowest = torch.where(torch.isinf(r["g"]), torch.full((), torch.finfo(F32).min), r["g"])
    o2, s2 = gdn.ops.linear_attn_fwd(*(t.to(cuda) for t in (r["q"], r["k"], r["v"], lowest)), initial_state=r["s0"].to(cuda))
    assert torch.equal(o, o2) and torch.equal(s, s2)


def test_column_slices_are_read_in_place(gdn, cuda):
    """q, k, v, g as column slices of one projection's rows, against dense copies: the same to the bit; slices off a
    16-byte boundary are copied first."""
    announce("linear attn slices")
    B, T, H, D = 2, 140, 2, 128
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn(B, T, 3 * H * D + 8 + H, generator=gen).to(BF).to(cuda)
    wide[..., -H:] = -wide[..., -H:].abs()
    for at in (0, 3):
        q, k, v = (wide[..., at + i * H * D: at + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
        g = wide[..., -H:]
        a = gdn.ops.linear_attn_fwd(q, k, v, g)
        b = gdn.ops.linear_attn_fwd(*(t.contiguous() for t in (q, k, v, g)))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        st = torch.randn(T, H, D, D, generator=gen).to(cuda)
        s1, s2 = st.clone(), st.clone()
        a = gdn.ops.linear_attn_step(q[0], k[0], v[0], g[0], s1)
        b = gdn.ops.linear_attn_step(*(t[0].contiguous() for t in (q, k, v, g)), s2)
        assert torch.equal(a, b) and torch.equal(s1, s2)


@pytest.mark.parametrize("T,H", [(50, 2), (400, 1), (2600, 1)])
def test_state_in_place(gdn, cuda, T, H):
    """final_state written over initial_state, in calls of one segment, one run and several."""
    announce(f"linear attn in place T={T}")
    d = L.inputs((2, T), H, H, 128, 128, T, BF, n_states=2, slow=0.1)
    args = [d[n].to(cuda) for n in ("q", "k", "v", "g")]
    s0 = d["s0"].to(cuda)
    o, s = gdn.ops.linear_attn_fwd(*args, initial_state=s0.clone())
    at = s0.clone()
    o2, s2 = gdn.ops.linear_attn_fwd(*args, initial_state=at, final_state=at)
    o3, none = gdn.ops.linear_attn_fwd(*args, initial_state=s0, output_final_state=False)
    torch.cuda.synchronize()
    assert s2 is at and none is None
    assert torch.equal(o, o2) and torch.equal(s, at) and torch.equal(o, o3)


def test_cut_anywhere_and_stepped_on(gdn, cuda):
    """A prompt, a second call from its state and then single steps give what one call gives."""
    announce("linear attn continued")
    d = L.inputs((1, 230), 2, 4, 128, 128, 31, F32, n_states=1)
    o_ref, s_ref, o_mag, s_mag = L.tokens(d["q"], d["k"], d["v"], d["g"], d["s0"])
    x = {n: d[n].to(cuda) for n in ("q", "k", "v", "g", "s0")}
    cut = lambda a, b: [x[n][:, a:b] for n in ("q", "k", "v", "g")]  # noqa: E731
    o1, s = gdn.ops.linear_attn_fwd(*cut(0, 75), initial_state=x["s0"])
    o2, s = gdn.ops.linear_attn_fwd(*cut(75, 220), initial_state=s)
    steps = [gdn.ops.linear_attn_step(*(t[:, 0] for t in cut(i, i + 1)), s).unsqueeze(1) for i in range(220, 230)]
    o = torch.cat([o1, o2, *steps], 1)
    torch.cuda.synchronize()
    assert L.within(o, o_ref, L.out_bound(o_ref, o_mag, F32, 230, 128)) <= 1
    assert L.within(s, s_ref, L.state_bound(s_mag, 230)) <= 1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nothing_leaks_from_tokens_that_are_not_seen(gdn, cuda, dtype, bad):
    """A NaN or an infinity in one token's v, k or q: the tokens before it and the other sequences keep their results to
    the bit, whole rows of theirs."""
    announce(f"linear attn non-finite {bad} {dtype}")
    cu = torch.tensor([0, 100, 230, 300], dtype=torch.int32, device=cuda)
    d = L.inputs((1, 300), 1, 2, 128, 128, 9, dtype, n_states=3)
    x = {n: d[n].to(cuda) for n in ("q", "k", "v", "g", "s0")}
    run = lambda y: gdn.ops.linear_attn_fwd(y["q"], y["k"], y["v"], y["g"], initial_state=x["s0"], cu_seqlens=cu)  # noqa: E731
    o, s = run(x)
    for name in ("v", "k", "q"):
        for t in (100, 117, 170, 229):
            y = dict(x)
            y[name] = x[name].clone()
            y[name][0, t, 0, 5] = bad
            o2, s2 = run(y)
            assert torch.equal(o2[:, :100], o[:, :100]) and torch.equal(o2[:, 230:], o[:, 230:])
            # (beside such a value the block's sums are taken token by token: in another order)
            before = (o2[:, 100:t].double() - o[:, 100:t].double()).abs()
            assert bool((before <= 2 * torch.finfo(dtype).eps * o[:, 100:t].double().abs() + 1e-5).all())
            assert not bool(torch.isfinite(o2[0, t, 0]).all())
            assert torch.equal(s2[[0, 2]], s[[0, 2]])
            if name == "v":  # one value column of one head
                assert bool(torch.isfinite(o2[0, :, 1]).all()) and bool(torch.isfinite(o2[0, :, 0, 6:]).all())
            if name == "q":
                assert torch.equal(s2, s) and torch.equal(o2[:, t + 1:], o[:, t + 1:])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,Hk,Hv,K,V", [(1, 1, 1, 64, 64), (3, 2, 4, 128, 64), (5, 1, 3, 64, 128), (64, 16, 16, 128, 128),
                                         (130, 4, 16, 128, 128)])
def test_step(gdn, cuda, B, Hk, Hv, K, V, dtype):
    announce(f"linear attn step B={B} {Hk}/{Hv} {K}x{V} {dtype}")
    d = L.inputs((B, 1), Hk, Hv, K, V, B, dtype, n_states=B)
    st = d["s0"].to(cuda)
    o = gdn.ops.linear_attn_step(*(d[n][:, 0].to(cuda) for n in ("q", "k", "v", "g")), st)
    torch.cuda.synchronize()
    o_ref, s_ref, o_mag, s_mag = L.tokens(d["q"], d["k"], d["v"], d["g"], d["s0"])
    # (the state's update: three roundings; the output: those and a sum of K products)
    c = (K + 4) * 2.0**-24
    assert L.within(st, s_ref, 4 * 2.0**-24 * s_mag) <= 1
    assert L.within(o.unsqueeze(1), o_ref, torch.finfo(dtype).eps / 2 * (o_ref.abs() + c * o_mag) + c * o_mag) <= 1


@pytest.mark.parametrize("B", [4, 150])
def test_step_slots(gdn, cuda, B):
    """Slots of a larger table: other rows stay, a slot outside the table or named before gives zeros."""
    announce(f"linear attn step slots B={B}")
    H, D, n = 2 if B < 100 else 16, 128, B + 5
    d = L.inputs((B, 1), H, H, D, D, B, BF, n_states=n)
    gen = torch.Generator().manual_seed(B)
    slots = torch.randperm(n, generator=gen)[:B]
    dead = [1, 3] if B < 100 else [1, 3, 70, 149]
    live = [b for b in range(B) if b not in dead]
    slots[1], slots[3] = -1, slots[0]
    if B > 100:
        slots[70], slots[149] = n, slots[66]
    st = d["s0"].to(cuda)
    o = gdn.ops.linear_attn_step(*(d[x][:, 0].to(cuda) for x in ("q", "k", "v", "g")), st, slots=slots.to(cuda))
    at = d["s0"][slots[live]].to(cuda)
    o2 = gdn.ops.linear_attn_step(*(d[x][live, 0].to(cuda) for x in ("q", "k", "v", "g")), at)
    torch.cuda.synchronize()
    want = d["s0"].to(cuda)
    want[slots[live].to(cuda)] = at
    assert torch.equal(o[live], o2) and torch.equal(st, want) and not bool(o[dead].any())


def test_graph_replays_and_streams(gdn, cuda):
    """A captured prompt call and step, replayed with eager work between, and calls on another stream: the eager results,
    to the bit, each time."""
    announce("linear attn graph")
    d = L.inputs((1, 900), 2, 2, 128, 128, 77, BF, n_states=1, slow=0.1)
    x = [d[n].to(cuda) for n in ("q", "k", "v", "g")]
    s0 = d["s0"].to(cuda)
    cu = torch.tensor([0, 900], dtype=torch.int32, device=cuda)
    o_ref, s_ref = gdn.ops.linear_attn_fwd(*x, initial_state=s0)
    step = [t[:, 7] for t in x]
    st_ref = s0.clone()
    refs = []
    for _ in range(3):
        refs.append((gdn.ops.linear_attn_step(*step, st_ref).clone(), st_ref.clone()))
    st = s0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, s = gdn.ops.linear_attn_fwd(*x, initial_state=s0, cu_seqlens=cu)
    torch.cuda.synchronize()
    assert torch.equal(o, o_ref) and torch.equal(s, s_ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = gdn.ops.linear_attn_fwd(*x, initial_state=s0, cu_seqlens=cu)
        y = gdn.ops.linear_attn_step(*step, st)
    for i in range(3):
        o.zero_()
        s.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, o_ref) and torch.equal(s, s_ref)
        assert torch.equal(y, refs[i][0]) and torch.equal(st, refs[i][1])
        gdn.ops.linear_attn_fwd(*(t.roll(1, 1) for t in x), initial_state=s0)
        torch.cuda.synchronize()


def test_rows_behind_the_last_sequence_stay(gdn, cuda):
    """A device table that ends before the batch's rows: the rows behind it are not written (the C ABI on outputs that the
    caller owns), and tables that run past the batch or overlap touch nothing outside it."""
    announce("linear attn tables")
    d = L.inputs((1, 200), 1, 2, 64, 64, 5, BF, n_states=3)
    q, k, v, g = (d[n].to(cuda) for n in ("q", "k", "v", "g"))
    s0 = d["s0"].to(cuda)
    nat = gdn._native
    ws = torch.empty(nat.lib().zlin_attn_workspace_bytes(1, 3, 200, 1, 2, 64, 64, 1), dtype=torch.uint8, device=cuda)

    def run(table):
        o = torch.full((200, 2, 64), 7.0, dtype=BF, device=cuda)
        s = torch.empty(3, 2, 64, 64, device=cuda)
        cu = torch.tensor(table, dtype=torch.int32, device=cuda)
        nat.call("zlin_attn_fwd", q.data_ptr(), 64, k.data_ptr(), 64, v.data_ptr(), 128, 1, g.data_ptr(), 2, 0, s0.data_ptr(),
                 s.data_ptr(), o.data_ptr(), cu.data_ptr(), 3, 1, 200, 1, 2, 64, 64, 0.125, ws.data_ptr(), ws.numel(),
                 torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return o, s

    o, s = run([0, 60, 60, 150])
    assert bool((o[150:] == 7).all())
    o_ref, s_ref, o_mag, s_mag = L.tokens(d["q"][:, :150], d["k"][:, :150], d["v"][:, :150], d["g"][:, :150], d["s0"], 0.125,
                                          [0, 60, 60, 150])
    assert L.within(o[:150].unsqueeze(0), o_ref, L.out_bound(o_ref, o_mag, BF, 150, 64)) <= 1
    assert L.within(s, s_ref, L.state_bound(s_mag, 150)) <= 1
    o, s = run([0, 60, 100, 10**6])  # (clamped to the batch's rows)
    o2, s2 = run([0, 60, 100, 200])
    assert torch.equal(o, o2) and torch.equal(s, s2)
    run([0, 200, 0, 200])
    run([-5, 3, 2, 1])


@pytest.mark.parametrize("Hk,Hv,K,V,n,dtype", [(8, 8, 64, 64, 36, BF), (2, 8, 128, 64, 66, BF), (8, 8, 128, 128, 33, BF),
                                               (4, 8, 64, 128, 70, BF), (3, 6, 128, 64, 48, F32)])
def test_packed_batches_that_fill_the_device(gdn, cuda, Hk, Hv, K, V, n, dtype):
    """Enough sequences and heads that one stays whole for many chunks: lengths of one chunk and less, of several, of so
    many that they are cut all the same; more and fewer than a wave's lanes of sequences; states carried in and out."""
    announce(f"linear attn batch of {n} {Hk}/{Hv} {K}x{V} {dtype}")
    gen = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 150, (n,), generator=gen).tolist()
    lengths[1], lengths[2], lengths[n // 2], lengths[-1] = 1100, 0, 640, 321
    cu = [0]
    for length in lengths:
        cu.append(cu[-1] + length)
    d = L.inputs((1, cu[-1]), Hk, Hv, K, V, n, dtype, n_states=n, slow=0.2)
    _check(gdn, cuda, d, cu, msg=f"batch of {n}")


@pytest.mark.parametrize("B,T,Hk,Hv,K,V", [(32, 333, 8, 8, 64, 64), (20, 260, 2, 32, 64, 64), (40, 200, 8, 8, 128, 64)])
def test_padded_batches_that_fill_the_device(gdn, cuda, B, T, Hk, Hv, K, V):
    """Batches of sequences of several chunks that are not cut."""
    announce(f"linear attn batch {B} x {T} {Hk}/{Hv} {K}x{V}")
    _check(gdn, cuda, L.inputs((B, T), Hk, Hv, K, V, B + T, BF, n_states=B, slow=0.2), msg=f"{B} x {T}")


@pytest.mark.parametrize("K,V,Hk", [(64, 64, 8), (128, 128, 8), (128, 64, 4)])
def test_nothing_leaks_in_batches_that_fill_the_device(gdn, cuda, K, V, Hk):
    """Infinities and NaN in q, k and v of a few tokens of a large batch: what does not see them keeps its bits."""
    announce(f"linear attn non-finite in a batch {Hk}/8 {K}x{V}")
    B, T, Hv = 40, 170, 8
    d = L.inputs((B, T), Hk, Hv, K, V, 5, BF, slow=0.1)
    x = {n: d[n].to(cuda) for n in ("q", "k", "v", "g")}
    o, s = gdn.ops.linear_attn_fwd(*x.values())
    seen = torch.zeros(B, T, Hv, dtype=torch.bool, device=cuda)
    y = {n: t.clone() for n, t in x.items()}
    y["v"][3, 150, 2, 5] = math.inf
    seen[3, 150:, 2] = True
    y["v"][4, 64, 7] = math.nan
    seen[4, 64:, 7] = True
    y["k"][5, 100, 0, 1] = math.nan
    seen[5, 100:, : Hv // Hk] = True
    y["q"][7, 20, 1] = math.inf
    seen[7, 20, Hv // Hk: 2 * (Hv // Hk)] = True
    o2, s2 = gdn.ops.linear_attn_fwd(*y.values())
    torch.cuda.synchronize()
    assert torch.equal(o[~seen], o2[~seen]) and bool(torch.isfinite(o2[~seen].float()).all())
    touched = torch.zeros(B, Hv, dtype=torch.bool, device=cuda)
    touched[3, 2] = touched[4, 7] = True
    touched[5, : Hv // Hk] = True
    assert torch.equal(s[~touched], s2[~touched])
    assert not bool(torch.isfinite(o2[4, 64:, 7].float()).any()) and not bool(torch.isfinite(o2[3, 150:, 2, 5].float()).any())

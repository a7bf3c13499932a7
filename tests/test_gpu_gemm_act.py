"""``ops.gemm_act`` (a projection with bias, activation and residual) against float64: sizes around its tiles and odd
ones, strides and alignments, every activation, bias types, in place on the residual, and the layer that it stands in
with linear attention."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import linear_testing as L
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ACTS = {None: lambda t: t, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu,
        "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}


def _data(cuda, M, N, K, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return [t.to(cuda) for t in (r(M, K).to(BF), (r(N, K) * K**-0.5).to(BF), r(N).to(BF), r(M, N).to(BF))]


def _check(y, x, w, bias, act, res):
    """|error|: fp32 sums of K products and the bias, 2^-24 of their sizes each, through an activation whose slope is at
    most 1.13 (the steepest, GELU's) and whose own evaluation is off by 2^-20 of its argument (an exponential of up to
    2^4, reciprocals, erf); the sum with the residual; and the result's rounding, 2^-8 of it."""
    t = x.double() @ w.double().T
    size = x.double().abs() @ w.double().abs().T
    if bias is not None:
        t, size = t + bias.double(), size + bias.double().abs()
    want = ACTS[act](t)
    err = 1.13 * (x.shape[1] + 2) * 2.0**-24 * size + 2.0**-20 * t.abs()
    if res is not None:
        want, err = want + res.double(), err + 2.0**-24 * (want.abs() + res.double().abs())
    bound = err + 2.0**-8 * (want.abs() + err)
    worst = float(((y.double() - want).abs() / bound.clamp_min(1e-300)).max())
    print(f"[errors] {worst:.3f} of the bound")
    assert worst <= 1, worst


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8, 8), (3, 5, 7), (16, 64, 64), (17, 72, 136), (63, 65, 66), (64, 64, 1000),
                                   (65, 130, 128), (128, 2056, 1024), (129, 257, 72), (200, 1024, 512), (257, 384, 192),
                                   (300, 520, 264), (1, 2056, 1024), (2, 1000, 4096), (33, 8, 2048), (512, 16, 640)])
def test_sizes(gdn, cuda, M, N, K):
    announce(f"gemm_act {M}x{N}x{K}")
    x, w, b, r = _data(cuda, M, N, K, M + N + K)
    _check(gdn.ops.gemm_act(x, w), x, w, None, None, None)
    _check(gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=r), x, w, b, "silu", r)


@pytest.mark.parametrize("M", [4, 150, 1000])
@pytest.mark.parametrize("act", list(ACTS))
def test_activations(gdn, cuda, act, M):
    announce(f"gemm_act {act} M={M}")
    x, w, b, r = _data(cuda, M, 264, 256, M)
    _check(gdn.ops.gemm_act(x, w, bias=b.float(), activation=act), x, w, b, act, None)
    # arguments of all sizes, also where the exponentials leave fp32's range
    x = x * torch.logspace(-3, 2.5, M, device=cuda)[:, None].to(BF)
    _check(gdn.ops.gemm_act(x, w, bias=b, activation=act, residual=r), x, w, b, act, r)


@pytest.mark.parametrize("M,N,K", [(5, 136, 256), (130, 264, 256), (700, 256, 128)])
def test_strides_and_alignment(gdn, cuda, M, N, K):
    """Operands and outputs as slices of wider buffers, on and off 16-byte boundaries; what lies beside the output stays."""
    announce(f"gemm_act strides {M}x{N}x{K}")
    gen = torch.Generator().manual_seed(M)
    r = lambda *s: torch.randn(*s, generator=gen).to(BF).to(cuda)  # noqa: E731
    for at, pad in ((0, 64), (8, 40), (1, 41), (3, 16), (4, 4)):
        x, w, res = r(M, K + pad + at)[:, at:at + K], (r(N, K + pad + at) * K**-0.5)[:, at:at + K], r(M, N + pad + at)[:, at:at + N]
        b = r(N + 1)[1:]
        wide = torch.full((M + 2, N + pad + at), 5.0, dtype=BF, device=cuda)
        out = wide[1:-1, at:at + N]
        got = gdn.ops.gemm_act(x, w, bias=b, activation="gelu", residual=res, out=out)
        assert got is out
        _check(out, x, w, b, "gelu", res)
        out.fill_(5.0)
        assert bool((wide == 5).all())
    xt = r(K, M).T  # columns apart: copied first
    _check(gdn.ops.gemm_act(xt, w), xt, w, None, None, None)


@pytest.mark.parametrize("M", [3, 200, 1500])
def test_residual_in_place(gdn, cuda, M):
    announce(f"gemm_act in place M={M}")
    x, w, b, r = _data(cuda, M, 520, 256, M)
    want = gdn.ops.gemm_act(x, w, bias=b, activation="relu", residual=r)
    y = r.clone()
    assert gdn.ops.gemm_act(x, w, bias=b, activation="relu", residual=y, out=y) is y
    assert torch.equal(y, want)


@pytest.mark.parametrize("M", [5, 70, 400])
def test_rows_do_not_see_one_another(gdn, cuda, M):
    """NaN and infinities in one row of x, or of w, stay in that row or column of y; no rows give no rows."""
    announce(f"gemm_act non-finite M={M}")
    x, w, b, r = _data(cuda, M, 200, 120, M)
    want = gdn.ops.gemm_act(x, w, bias=b, residual=r)
    for bad in (math.nan, math.inf):
        x2, w2 = x.clone(), w.clone()
        x2[M // 2, 119] = bad
        w2[199, 0] = bad
        y = gdn.ops.gemm_act(x2, w2, bias=b, residual=r)
        keep = torch.ones(M, dtype=torch.bool, device=cuda)
        keep[M // 2] = False
        assert torch.equal(y[keep, :199], want[keep, :199])
        assert not bool(torch.isfinite(y[M // 2]).any()) and not bool(torch.isfinite(y[:, 199]).any())
    assert gdn.ops.gemm_act(x[:0], w, bias=b).shape == (0, 200)


def test_graph_replays(gdn, cuda):
    announce("gemm_act graph")
    data = [_data(cuda, M, 2056, 1024, M) for M in (4, 900)]
    want = [gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=r) for x, w, b, r in data]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=r) for x, w, b, r in data]
    for _ in range(3):
        for y in got:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        gdn.ops.gemm_act(data[1][0].flip(0), data[1][1])
        torch.cuda.synchronize()


def test_a_layer_of_linear_attention(gdn, cuda):
    """The operators as a mixer layer runs them: q, k, v and gate from one projection with SiLU, linear attention, gated
    norm, output projection onto the residual stream -- over a prompt and on by single steps, against float64."""
    announce("linear attention layer")
    H, D, hidden, T, more = 2, 128, 256, 150, 3
    gen = torch.Generator().manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = r(T + more, hidden).to(BF)
    w_in, w_out = (r(4 * H * D, hidden) * hidden**-0.5).to(BF), (r(hidden, H * D) * (H * D) ** -0.5).to(BF)
    b_in, nw = (0.1 * r(4 * H * D)).to(BF), (1 + 0.1 * r(D)).to(BF)
    g = torch.tensor([-0.3, -0.01])
    c = {n: t.to(cuda) for n, t in dict(x=x, w_in=w_in, w_out=w_out, b_in=b_in, nw=nw, g=g).items()}
    ops = gdn.ops

    def layer(rows, state):
        n = len(rows)
        z = ops.gemm_act(rows, c["w_in"], bias=c["b_in"], activation="silu").view(n, 4, H, D)
        if n > 1:
            o, state = ops.linear_attn_fwd(z[None, :, 0], z[None, :, 1], z[None, :, 2], c["g"])
            o = o[0]
        else:
            o = ops.linear_attn_step(z[:, 0], z[:, 1], z[:, 2], c["g"], state)
        y, _ = ops.gated_rmsnorm(o, z[:, 3].contiguous(), c["nw"], eps=1e-5)
        return ops.gemm_act(y.view(n, H * D), c["w_out"], residual=rows), state

    ys = []
    y, state = layer(c["x"][:T], None)
    ys.append(y)
    for t in range(T, T + more):
        y, state = layer(c["x"][t:t + 1], state)
        ys.append(y)
    got = torch.cat(ys)
    torch.cuda.synchronize()
    rnd = lambda t: t.to(BF).double()  # noqa: E731  -- the rounding points of the layer
    z = rnd(F.silu(x.double() @ w_in.double().T + b_in.double())).view(T + more, 4, H, D)
    o = rnd(L.tokens(z[None, :, 0], z[None, :, 1], z[None, :, 2], g)[0][0])
    n = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-5) * nw.double()
    y = rnd(n * F.silu(z[:, 3])).view(T + more, H * D)
    want = y @ w_out.double().T + x.double()
    # the kernels round at the same four points; where a value lies next to a border one may go the other way, a step
    # (2^-7 of it): of the mixer's terms, at worst 4 x 2^-7 in 2-norm, and the result's own rounding of the whole
    err, mixer = (got.cpu().double() - want).norm(), (want - x.double()).norm()
    print(f"[errors] {float(err / mixer):.2e} of the mixer's part")
    assert float(err) <= 4 * 2.0**-7 * float(mixer) + 2.0**-8 * float(want.norm())


def test_columns_beside_one_another(gdn, cuda):
    """x, the residual and y as columns of one buffer's rows; the same columns are refused."""
    announce("gemm_act columns of one buffer")
    M, N, K = 70, 64, 128
    x, w, b, r = _data(cuda, M, N, K, 9)
    buf = torch.cat([x, r, torch.zeros_like(r)], 1)
    y = buf[:, K + N:]
    gdn.ops.gemm_act(buf[:, :K], w, bias=b, activation="silu", residual=buf[:, K: K + N], out=y)
    torch.cuda.synchronize()
    assert torch.equal(y, gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=r))
    assert torch.equal(buf[:, :K], x) and torch.equal(buf[:, K: K + N], r)
    for bad in (buf[:, :N], buf[:, K - 8: K - 8 + N], buf[:, K + 8: K + 8 + N]):
        with pytest.raises(RuntimeError, match="overlap"):
            gdn.ops.gemm_act(buf[:, :K], w, residual=buf[:, K: K + N], out=bad)


@pytest.mark.parametrize("M,N,K", [(1100, 17, 264), (1100, 17, 261), (2000, 8, 512), (900, 72, 520), (513, 130, 333), (40, 3, 2050),
                                   (70, 600, 130), (129, 300, 190)])
def test_few_columns_and_odd_rows(gdn, cuda, M, N, K):
    """Tall products of few columns (fewer column tiles than XCDs), rows off 16-byte boundaries, K behind its last block."""
    announce(f"gemm_act tall {M}x{N}x{K}")
    x, w, b, r = _data(cuda, M, N, K, M + N + K)
    _check(gdn.ops.gemm_act(x, w, bias=b, activation="relu", residual=r), x, w, b, "relu", r)
    wide = torch.full((M, K + 3), float("nan"), dtype=BF, device=cuda)  # rows 2 bytes off, beside values that nobody may use
    wide[:, 1: 1 + K] = x
    _check(gdn.ops.gemm_act(wide[:, 1: 1 + K], w), x, w, None, None, None)

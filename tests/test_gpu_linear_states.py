"""Linear attention's states where little is left of them: strong decays behind which no token adds anything. What is left is
held to float64 relative to its own size, not to that of what it was (bounds: ``linear_testing``)."""

from __future__ import annotations

import pytest
import torch

import linear_testing as L
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
SUMS = [-0.1, -0.6, -2.0, -4.0, -8.0, -12.0, -16.0, -30.0]  # of a chunk's log decays, by head


def _quiet(B, T, Hk, Hv, K, V, seed, dtype):
    """64 tokens as usual, then none with values: 128 whose decays sum to ``SUMS`` a chunk of 64, the others slow."""
    d = L.inputs((B, T), Hk, Hv, K, V, seed, dtype)
    d["v"][:, 64:] = 0
    share = torch.rand(B, T, Hv, generator=torch.Generator().manual_seed(seed + 1)) + 0.1
    g = torch.full((B, T, Hv), -0.05 / 64)
    for lo in (64, 128):
        w = share[:, lo: lo + 64]
        g[:, lo: lo + 64] = torch.tensor(SUMS).repeat(Hv // len(SUMS)) * w / w.sum(1, keepdim=True)
    d["g"] = g
    return d


SMALLEST = 2.0**-126  # fp32's least normal number: exp(-150) times anything of a test's size lies below, and below it a
# value has no 24 bits (and a matrix product may take it as zero): nothing smaller is held to a relative bound


def _hold(gdn, cuda, d, dtype):
    T, K = d["q"].shape[1], d["q"].shape[3]
    o, s = gdn.ops.linear_attn_fwd(*(d[n].to(cuda) for n in ("q", "k", "v", "g")))
    torch.cuda.synchronize()
    o_ref, s_ref, o_mag, s_mag = L.tokens(d["q"], d["k"], d["v"], d["g"])
    eo = L.within(o, o_ref, L.out_bound(o_ref, o_mag, dtype, T, K) + SMALLEST)
    es = L.within(s, s_ref, L.state_bound(s_mag, T) + SMALLEST)
    print(f"[errors] outputs {eo:.3f}, states {es:.3f} of their bounds")
    assert eo <= 1 and es <= 1, (eo, es)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,Hk,Hv,K,V", [(32, 192, 8, 8, 64, 64), (40, 192, 8, 8, 128, 64), (2, 200, 2, 8, 128, 128),
                                           (1, 1280, 8, 64, 64, 128)])
def test_what_is_left_behind_strong_decays(gdn, cuda, B, T, Hk, Hv, K, V, dtype):
    """Sequences walked whole by 8 and by 4 waves, in segments of one chunk and of five."""
    announce(f"linear attn quiet tail {B} x {T} {Hk}/{Hv} {K}x{V} {dtype}")
    d = _quiet(B, T, Hk, Hv, K, V, B + T, dtype)
    _hold(gdn, cuda, d, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_quiet_prompt_and_quiet_steps_agree(gdn, cuda, dtype):
    """The same quiet tokens as one prompt and as single steps from the same state: the same state, within its bound."""
    announce(f"linear attn quiet steps {dtype}")
    B, T, H = 32, 192, 8
    d = {n: t.to(cuda) if t is not None else None for n, t in _quiet(B, T, H, H, 64, 64, 3, dtype).items()}
    _, s = gdn.ops.linear_attn_fwd(*(d[n] for n in ("q", "k", "v", "g")))
    _, at = gdn.ops.linear_attn_fwd(*(d[n][:, :64] for n in ("q", "k", "v", "g")))
    for t in range(64, T):
        gdn.ops.linear_attn_step(*(d[n][:, t] for n in ("q", "k", "v", "g")), at)
    torch.cuda.synchronize()
    mag = L.tokens(*(d[n] for n in ("q", "k", "v", "g")))[3]
    assert L.within(s, at.double().cpu(), 2 * L.state_bound(mag, T)) <= 1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,H", [(2, 150, 2), (40, 128, 8)])
@pytest.mark.parametrize("low", [float("-inf"), -150.0, -20.0])
def test_slow_tokens_behind_many_fast_ones(gdn, cuda, low, B, T, H, dtype):
    """Dozens of resets, or of decays nearly as strong, in a chunk and a run of slow tokens behind them: the weights of those
    among one another are as exact as anywhere. Keys and queries near one direction, so that every token has its part in an
    output, values of both signs, so that outputs are smaller than their parts."""
    announce(f"linear attn {low} and slow, {B} x {T} {H} {dtype}")
    d = L.inputs((B, T), H, H, 64, 64, 17, dtype)
    one = torch.nn.functional.normalize(torch.randn(64, generator=torch.Generator().manual_seed(1)), dim=0)
    for n in ("q", "k"):
        d[n] = torch.nn.functional.normalize(one + 0.3 * d[n].float(), dim=-1).to(dtype)
    at = torch.arange(T) % 64
    d["g"] = torch.where((at < 48)[None, :, None], torch.full((), low), 0.05 * d["g"])
    _hold(gdn, cuda, d, dtype)

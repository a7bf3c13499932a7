"""Linear attention repeats itself to the bit, whatever the device's memory and LDS held before: between calls other kernels
fill the LDS and the allocator's free blocks (where outputs and workspaces come from) hold NaN."""

from __future__ import annotations

import pytest
import torch

import linear_testing as L
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lead,Hk,Hv,K,V,cu", [((2, 64), 4, 4, 128, 128, None), ((1, 1000), 4, 4, 128, 128, None),
                                               ((1, 700), 2, 8, 64, 64, [0, 64, 65, 65, 400, 650]),
                                               ((36, 190), 8, 8, 128, 64, None), ((3, 1), 1, 2, 64, 128, None)])
def test_calls_repeat_to_the_bit(gdn, cuda, lead, Hk, Hv, K, V, cu, dtype):
    announce(f"linear attn repeats {lead} {Hk}/{Hv} {K}x{V} {dtype}")
    n = lead[0] if cu is None else len(cu) - 1
    d = {x: t.to(cuda) for x, t in L.inputs(lead, Hk, Hv, K, V, 4, dtype, n_states=n).items()}
    table = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=cuda)
    rows = lead[1] if cu is None else cu[-1]
    x, w = (torch.randn(s, 2048, device=cuda).to(BF) * 1e4 for s in (900, 640))
    first = None
    for i in range(12):
        if i % 2:  # (free blocks of the sizes that the call asks for)
            size = gdn._native.lib().zlin_attn_workspace_bytes(int(cu is not None), n, lead[1], Hk, Hv, K, V, 0 if dtype == F32 else 1)
            dirt = [torch.full_like(d["v"], float("nan")), torch.full((n, Hv, V, K), float("nan"), device=cuda),
                    torch.full((max(size, 1),), 0xFF, dtype=torch.uint8, device=cuda)]
            del dirt
        if i % 3:
            gdn.ops.gemm_act(x, w)
        o, s = gdn.ops.linear_attn_fwd(d["q"], d["k"], d["v"], d["g"], initial_state=d["s0"], cu_seqlens=table)
        o = o[:, :rows].clone()
        if first is None:
            first = o, s.clone()
        assert torch.equal(o, first[0]) and torch.equal(s, first[1]), i

"""Linear attention's C entry on device tables that are no packed batch's (overlapping, decreasing, running past the rows):
nothing outside its outputs and its workspace is written, and rows and states of no sequence stay or come through."""

from __future__ import annotations

import pytest
import torch

import linear_testing as L
from gdn_testing import announce

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
PAD = 1 << 16  # bytes kept before and behind each buffer that the call may write


class _Guarded:
    """A tensor in the middle of a buffer of its own, whose other bytes have to stay."""

    def __init__(self, shape, dtype, device, fill):
        n = torch.Size(shape).numel() * dtype.itemsize
        self.raw = torch.full((2 * PAD + n,), 0x5A, dtype=torch.uint8, device=device)
        self.t = self.raw[PAD: PAD + n].view(dtype).view(shape)
        self.t.fill_(fill)

    def kept(self) -> bool:
        n = self.t.numel() * self.t.element_size()
        return bool((self.raw[:PAD] == 0x5A).all()) and bool((self.raw[PAD + n:] == 0x5A).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,table", [(200, [0, 200, 0, 200]), (200, [-5, 3, 2, 1]), (200, [150, 10**6, 0, 77]),
                                     (700, [0, 700, 0, 700, 0, 700]), (64, [64, 64, 0, 0])])
def test_tables_touch_nothing_outside(gdn, cuda, T, table, dtype):
    announce(f"linear attn table {table} of {T} rows, {dtype}")
    n, Hv, D, nat = len(table) - 1, 2, 64, gdn._native
    d = L.inputs((1, T), 1, Hv, D, D, 5, dtype, n_states=n)
    q, k, v, g, s0 = (d[x].to(cuda) for x in ("q", "k", "v", "g", "s0"))
    code = 0 if dtype == F32 else 1
    size = nat.lib().zlin_attn_workspace_bytes(1, n, T, 1, Hv, D, D, code)
    o, s = _Guarded((T, Hv, D), dtype, cuda, 7.0), _Guarded((n, Hv, D, D), F32, cuda, 9.0)
    ws = _Guarded((max(size, 16),), torch.uint8, cuda, 0xFF)  # (as floats: NaN)
    cu = torch.tensor(table, dtype=torch.int32, device=cuda)
    nat.call("zlin_attn_fwd", q.data_ptr(), D, k.data_ptr(), D, v.data_ptr(), Hv * D, code, g.data_ptr(), Hv, 0, s0.data_ptr(),
             s.t.data_ptr(), o.t.data_ptr(), cu.data_ptr(), n, 1, T, 1, Hv, D, D, 0.125, ws.t.data_ptr(), size,
             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert o.kept() and s.kept() and ws.kept()
    rows = torch.zeros(T, dtype=torch.bool)
    bounds = []  # as they are clamped
    for i in range(n):
        lo = min(max(table[i], 0), T)
        bounds.append((lo, min(max(table[i + 1], lo), T)))
    for i, (lo, hi) in enumerate(bounds):
        rows[lo:hi] = True
        # an empty sequence: its state comes through (what sequences that overlap give is not specified)
        if hi == lo and sum(b - a for a, b in bounds) <= T:
            assert torch.equal(s.t[i], s0[i]), i
    assert bool((o.t.cpu()[~rows] == 7).all())
    if table[0] == -5:  # one sequence of rows 0 .. 2
        o_ref, s_ref, o_mag, s_mag = L.tokens(*(d[x][:, :3] for x in ("q", "k", "v", "g")), d["s0"], 0.125, [0, 3])
        assert L.within(o.t[None, :3], o_ref, L.out_bound(o_ref, o_mag, dtype, 3, D)) <= 1
        assert L.within(s.t[:1], s_ref, L.state_bound(s_mag, 3)) <= 1

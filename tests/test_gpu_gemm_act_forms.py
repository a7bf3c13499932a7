"""``ops.gemm_act`` in each of its kernels, by sizes that take it (asserted), against float64: remainders of rows, columns and K,
outputs whose rows allow accesses of 8, 4 and 1 elements, columns beside the output, the residual in place, operands
among values that nobody may use. Bounds: ``test_gpu_gemm_act``."""

from __future__ import annotations

import pytest
import torch

from gdn_testing import announce
from test_gemm_act_forms import ANY64, ANY128, FOLD, SPLIT16, SPLIT32, TILE64, TILE256, WIDE, form
from test_gpu_gemm_act import _check, _data

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

CASES = [(SPLIT16, 9, 77, 1160), (SPLIT32, 70, 1100, 520), (TILE64, 700, 650, 328), (FOLD, 3585, 1025, 72),
         (FOLD, 3611, 1032, 200), (FOLD, 3001, 1296, 328), (WIDE, 4103, 1000, 328), (WIDE, 8247, 390, 72),
         (WIDE, 8300, 512, 136), (TILE256, 8913, 1281, 200), (TILE256, 4917, 2500, 72), (TILE256, 5000, 2560, 328),
         (SPLIT16, 9, 77, 1161), (SPLIT32, 70, 1100, 521), (ANY64, 700, 650, 67), (ANY128, 2549, 777, 201),
         (ANY128, 3585, 520, 333), (ANY128, 1587, 1300, 64 * 3 + 1)]


@pytest.mark.parametrize("f,M,N,K", CASES)
def test_form(gdn, cuda, f, M, N, K):
    announce(f"gemm_act form {f} {M}x{N}x{K}")
    assert form(gdn._native, M, N, K, K % 8 == 0)[0] == f
    x, w, b, r = _data(cuda, M, N, K, M + N + K)
    y = gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=r)
    _check(y, x, w, b, "silu", r)
    _check(gdn.ops.gemm_act(x, w, bias=b.float()), x, w, b, None, None)
    at = r.clone()
    assert gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=at, out=at) is at and torch.equal(at, y)
    for off, pad in ((8, 8 - (8 + N) % 8), (4, 4 - N % 4), (1, 2)):  # rows that start every 16, 8 and 2 bytes
        wide = torch.full((M + 2, off + N + pad), 5.0, dtype=BF, device=cuda)
        out = wide[1:-1, off: off + N]
        res = torch.full((M, off + N + pad), float("nan"), dtype=BF, device=cuda)[:, off: off + N]
        res.copy_(r)
        gdn.ops.gemm_act(x, w, bias=b, activation="silu", residual=res, out=out)
        assert torch.equal(out, y), (off, pad)
        out.fill_(5.0)
        assert bool((wide == 5).all())


@pytest.mark.parametrize("f,M,N,K", [c for c in CASES if c[3] % 8 == 0])
def test_form_reads_its_operands_alone(gdn, cuda, f, M, N, K):
    """x and w as columns of rows whose other columns, and the rows around them, are NaN; the forms of direct loads."""
    announce(f"gemm_act form {f} {M}x{N}x{K} among NaN")
    x, w, _, _ = _data(cuda, M, N, K, M + N + K)
    among = []
    for t in (x, w):
        wide = torch.full((t.shape[0] + 2, K + 24), float("nan"), dtype=BF, device=cuda)
        wide[1:-1, 8: 8 + K] = t
        among.append(wide[1:-1, 8: 8 + K])
    assert form(gdn._native, M, N, K)[0] == f and among[0].data_ptr() % 16 == 0 and among[1].stride(0) % 8 == 0
    y = gdn.ops.gemm_act(*among)
    _check(y, x, w, None, None, None)
    assert torch.equal(y, gdn.ops.gemm_act(x, w))

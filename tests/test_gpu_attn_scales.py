"""Attention at the ends of the scale's range: no scale, scales as small as scores are large, scales that have no
finite product with log2 e (bounds: ``attn_testing``)."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

import attn_testing as A
from gdn_testing import announce

BF, F32 = torch.bfloat16, torch.float32


def _inputs(T, D, dtype, size):
    """Queries and keys of `size`: their products are of size^2."""
    g = torch.Generator().manual_seed(61)
    q, k, v = (A.randn(g, T, h, D) for h in (4, 2, 2))
    return (size * q).to(dtype), (size * k).to(dtype), v.to(dtype)


# T, Tq, D, window; rows of a workgroup, whether several share their keys
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,Tq,D,window,rows,shared", [(4500, 4500, 128, 100, 128, False), (400, 400, 64, None, 32, False),
                                                       (2500, 8, 128, None, 32, True)])
@pytest.mark.parametrize("scale,size", [(0.0, 1e16), (1e-32, 3e15), (-1e-32, 3e15), (1e-36, 3e17), (1e-40, 1e18), (1.0, 0.3)])
def test_scores_of_any_size(gdn, cuda, scale, size, T, Tq, D, window, rows, shared, dtype):
    """Products of up to 1e37 by scales down to zero, over sequences in each form, and for one token."""
    announce(f"attention, scale {scale} size {size} T {T}/{Tq} D {D} {dtype}")
    form = (ctypes.c_int64 * 2)()
    gdn.ops._native.call("zgdn_window_fwd_form", 0, 1, Tq, T, 4, 2, D, window or 0, 0, int(dtype == BF), form)
    assert (form[0], form[1] > 1) == (rows, shared)
    q, k, v = _inputs(T, D, dtype, size)
    q = q[-Tq:]
    o = gdn.window_attn_fwd(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), window=window, scale=scale)[0].cpu()
    x = gdn.window_attn_step(q[-1:].to(cuda), k[None].to(cuda), v[None].to(cuda), torch.tensor([T], dtype=torch.int32, device=cuda),
                             window=window, scale=scale).cpu()
    torch.cuda.synchronize()
    at = torch.unique(torch.cat([torch.arange(min(Tq, 4)), torch.arange(0, Tq, 97), torch.arange(max(0, Tq - 4), Tq)]))
    want, sizes, slip = A.attend(q[at], k, v, T - Tq + at, window=window, scale=scale)
    # the scale itself and its product with log2 e are rounded to float32: each half a step, of 2^-149 below 2^-126
    terms = float(q.double().abs().amax() * k.double().abs().amax()) * D
    bound = A.attend_bound(want, sizes, slip + 2 * max(2.0**-24 * abs(scale), 2.0**-150) * terms, dtype, T)
    assert A.within(o[at], want, bound) <= 1
    assert A.within(x[0], want[-1], bound[-1]) <= 1


def test_scales_without_a_product_are_refused():
    native = importlib.import_module("zonos3-mini_amd._native")
    at = lambda n: ctypes.c_void_p((1 << 32) + (n << 28))  # noqa: E731  (never read: calls of nothing)
    for scale in (2.4e38, -3.4e38):
        with pytest.raises(RuntimeError, match="scale"):
            native.call("zattn_window_fwd", at(0), 256, at(1), 128, at(2), 128, 1, at(3), None, None, 0, 1, 0, 9, 4, 2, 64, 0, 0,
                        scale, None, 0, None)
        with pytest.raises(RuntimeError, match="scale"):
            native.call("zattn_window_step", at(0), 256, at(1), 128, at(2), 128, 1, at(4), None, 9, 1, 9, at(3), 0, 4, 2, 64, 0, 0,
                        scale, None, 0, None)

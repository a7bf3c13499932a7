"""The attention sublayer's operators without a GPU: the header's entry points, what they refuse (before any launch), the host
layer's refusals, the registered operators."""

from __future__ import annotations

import ctypes
import importlib
import re
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

ROOT = Path(__file__).resolve().parents[1]


def _at(n):  # (never read: every call below is refused)
    return ctypes.c_void_p((1 << 32) + (n << 28))


P = _at(0)
ODD = ctypes.c_void_p((1 << 32) + 8)


@pytest.fixture(scope="module")
def native():
    return importlib.import_module("zonos3-mini_amd._native")


def test_header_and_library_agree(native):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "zonos3_attn.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(zattn_\w+)\s*\(", text))
    assert names == set(native.ATTN)
    for n in names:
        assert hasattr(native.lib(), n)
        declared = re.search(rf"\b{n}\s*\(([^)]*)\)", text).group(1)
        assert len(declared.split(",")) == len(native.ATTN[n][1]), n


def _refused(native, name, args, cases):
    for over, match in cases:
        assert set(over) <= set(args)
        with pytest.raises(RuntimeError, match=match):
            native.call(name, *{**args, **over}.values())


def test_qk_norm_rope_refuses(native):
    args = dict(q=P, q_ld=1024, k=_at(1), k_ld=256, v=_at(2), v_ld=256, dtype=1, pos=_at(3), pos32=0, freq=_at(4), freq32=0,
                qw=_at(5), kw=_at(5), w_dtype=1, eps=1e-6, inter=0, q_out=_at(6), k_out=_at(7), kc=_at(8), kc_ld=256,
                vc=_at(9), vc_ld=256, rows=_at(10), n_rows=64, n=5, Hq=8, Hk=2, D=128, R=128, stream=None)
    _refused(native, "zattn_qk_norm_rope", args, [
        (dict(n=-1), "bad sizes"), (dict(Hq=0), "bad sizes"), (dict(Hk=0), "bad sizes"), (dict(n_rows=-1), "bad sizes"),
        (dict(D=96), "D=96"), (dict(R=24), "R=24"), (dict(R=144), "R=144"), (dict(R=-16), "R=-16"), (dict(dtype=2), "dtype code 2"),
        (dict(w_dtype=9), "dtype code 9"), (dict(rows=None), "go together"), (dict(kc=None), "go together"),
        (dict(v=None), "go together"), (dict(vc=None), "go together"), (dict(q=None), "null"), (dict(freq=None), "null"),
        (dict(q_out=None), "null"), (dict(pos=None), "null"), (dict(q_ld=1020), "row strides"), (dict(k_ld=128), "row strides"),
        (dict(v_ld=260), "row strides"), (dict(kc_ld=1 << 23), "row strides"), (dict(vc_ld=8), "row strides"), (dict(q=ODD), "16-byte"),
        (dict(qw=ODD), "16-byte"), (dict(vc=ODD), "16-byte"), (dict(pos=ctypes.c_void_p((1 << 34) + 4)), "boundary"),
        (dict(rows=ctypes.c_void_p((1 << 34) + 4)), "boundary"), (dict(q_out=P), "overlaps"), (dict(k_out=_at(6)), "overlaps"),
        (dict(kc=_at(1)), "overlaps"), (dict(vc=_at(8)), "overlaps"), (dict(n=1 << 27), "n_tokens=")])
    # slices of a joint cache do not overlap, nor does a call of no tokens read anything
    assert native.lib().zattn_qk_norm_rope(*{**args, "n": 0}.values()) == native.OK
    _refused(native, "zattn_qk_norm_rope", {**args, "kc_ld": 512, "vc_ld": 512}, [(dict(vc=ctypes.c_void_p(_at(8).value + 256)), "overlaps")])


def test_window_fwd_refuses(native):
    args = dict(q=P, q_ld=1024, k=_at(1), k_ld=256, v=_at(2), v_ld=256, dtype=1, o=_at(3), cu_q=None, cu_k=None, n_seqs=0, B=2,
                Tq=100, Tk=130, Hq=8, Hk=2, D=128, window=64, sinks=4, scale=1.0, ws=None, ws_bytes=0, stream=None)
    _refused(native, "zattn_window_fwd", args, [
        (dict(B=0), "bad sizes"), (dict(Tq=-1), "bad sizes"), (dict(window=-1), "bad sizes"), (dict(sinks=-1), "bad sizes"),
        (dict(Hk=3), "multiple"), (dict(D=256), "D=256"), (dict(dtype=5), "dtype code 5"), (dict(cu_q=_at(4)), "go together"),
        (dict(cu_q=_at(4), cu_k=_at(5), n_seqs=2), "B == 1"), (dict(cu_q=_at(4), cu_k=_at(5), B=1), "n_seqs"),
        (dict(q=None), "null"), (dict(v=None), "null"), (dict(o=None), "null"), (dict(q_ld=1023), "row strides"),
        (dict(k_ld=248), "row strides"), (dict(v_ld=1 << 23), "row strides"), (dict(k=ODD), "16-byte"), (dict(o=P), "overlaps"),
        (dict(o=ctypes.c_void_p(_at(2).value + 512)), "overlaps"), (dict(B=1 << 12, Tq=1 << 20), "rows"),
        (dict(cu_q=ctypes.c_void_p(_at(4).value + 2), cu_k=_at(5), B=1, n_seqs=2), "4-byte"),
        (dict(ws=ODD), "16-byte"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale")])
    assert native.lib().zattn_window_fwd(*{**args, "Tq": 0}.values()) == native.OK


def test_window_step_refuses(native):
    size = native.lib().zattn_window_step_workspace_bytes
    for bad in ((-1, 64, 8, 2, 128, 0, 0, 1), (2, -1, 8, 2, 128, 0, 0, 1), (2, 64, 8, 3, 128, 0, 0, 1), (2, 64, 8, 2, 96, 0, 0, 1),
                (2, 64, 8, 2, 128, -1, 0, 1), (2, 64, 8, 2, 128, 0, 0, 2), (2, 1 << 31, 8, 2, 128, 0, 0, 1)):
        assert size(*bad) == 0
    need = size(2, 65536, 8, 2, 128, 0, 0, 1)
    assert 0 < need and size(2, 65536, 8, 2, 128, 100, 4, 1) < need
    args = dict(q=P, q_ld=1024, kc=_at(1), kc_ld=256, vc=_at(2), vc_ld=256, dtype=1, lengths=_at(3), pages=_at(4), page_size=64,
                n_pages=1024, n_rows=1 << 17, o=_at(5), B=2, Hq=8, Hk=2, D=128, window=0, sinks=0, scale=1.0, ws=_at(6),
                ws_bytes=need, stream=None)
    _refused(native, "zattn_window_step", args, [
        (dict(B=-1), "bad sizes"), (dict(n_rows=-64), "bad sizes"), (dict(sinks=-2), "bad sizes"), (dict(Hq=7), "multiple"),
        (dict(D=32), "D=32"), (dict(dtype=4), "dtype code 4"), (dict(page_size=48), "power of two"), (dict(page_size=0), "power of two"),
        (dict(n_rows=100), "power of two"), (dict(pages=None), "one a stream"), (dict(pages=None, n_pages=1, n_rows=100), "one a stream"),
        (dict(n_pages=1 << 25), "positions a stream"), (dict(lengths=None), "null"), (dict(vc=None), "null"), (dict(kc_ld=250), "row strides"),
        (dict(vc_ld=128), "row strides"), (dict(q_ld=1 << 23), "row strides"), (dict(kc=ODD), "16-byte"), (dict(ws=ODD), "16-byte"),
        (dict(pages=ctypes.c_void_p(_at(4).value + 2)), "4-byte"), (dict(ws=None), "workspace"), (dict(ws_bytes=need - 1), "workspace"),
        (dict(o=P), "overlap"), (dict(ws=_at(1)), "overlap"), (dict(ws=_at(5)), "overlap"), (dict(scale=float("-inf")), "scale")])
    assert native.lib().zattn_window_step(*{**args, "B": 0}.values()) == native.OK


def test_host_layer_refuses_cpu_tensors(gdn):
    q, n = torch.zeros(1, 2, 1, 128), torch.zeros(1, 2, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gdn.qk_norm_rope(q, q, n, torch.zeros(64))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gdn.window_attn_fwd(q, q, q)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gdn.window_attn_step(q[0], q, q, torch.ones(2, dtype=torch.int32))
    for call in (lambda: gdn.qk_norm_rope(None, q, n, q), lambda: gdn.window_attn_fwd(None, q, q),
                 lambda: gdn.window_attn_step(None, q, q, n)):
        with pytest.raises(RuntimeError, match="expected a tensor"):
            call()
    for call in (lambda x: gdn.qk_norm_rope(x, x, n, torch.zeros(64)), lambda x: gdn.window_attn_fwd(x, x, x)):
        with pytest.raises(RuntimeError, match="not supported"):
            call(q.half())


def test_registered_operators(gdn):
    z = torch.ops.zgdn
    ops = importlib.import_module("zonos3-mini_amd.torch_ops")
    names = {"qk_norm_rope", "qk_norm_rope_cache", "window_attn_fwd", "window_attn_step"}
    assert names <= set(ops.OPERATORS)
    writes = lambda n: {a.name for a in getattr(z, n).default._schema.arguments  # noqa: E731
                        if a.alias_info is not None and a.alias_info.is_write}
    assert {n: writes(n) for n in names if writes(n)} == {"qk_norm_rope_cache": {"k_cache", "v_cache"}}
    with FakeTensorMode():
        q, k = torch.empty(3, 70, 8, 128, dtype=torch.bfloat16), torch.empty(3, 70, 2, 128, dtype=torch.bfloat16)
        at, f, c = torch.empty(3, 70, dtype=torch.long), torch.empty(64), torch.empty(9, 64, 2, 128, dtype=torch.bfloat16)
        a, b = z.qk_norm_rope(q, k, at, f)
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == b.dtype == q.dtype
        assert z.qk_norm_rope_cache(q, k, k, at, f, c, c, at).shape == q.shape
        assert z.window_attn_fwd(q, k, k, 5).shape == q.shape
        assert z.window_attn_step(q[0], c, c, at[0].int(), None, 0, None, at.int()[:, :4]).shape == (70, 8, 128)


@pytest.mark.gpu
def test_operators_run_what_the_direct_calls_run(gdn, cuda):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda)  # noqa: E731
    z = torch.ops.zgdn
    q, k, v = r(1, 90, 4, 64), r(1, 90, 2, 64), r(1, 90, 2, 64)
    at, f = torch.arange(90, device=cuda)[None], torch.rand(32, generator=g).to(cuda)
    assert all(torch.equal(x, y) for x, y in zip(gdn.qk_norm_rope(q, k, at, f), z.qk_norm_rope(q, k, at, f)))
    assert torch.equal(gdn.window_attn_fwd(q, k, v, window=20, sinks=2), z.window_attn_fwd(q, k, v, 20, 2))
    kc, vc = r(8, 16, 2, 64), r(8, 16, 2, 64)
    rows = torch.randperm(128, generator=g)[:90][None].to(cuda)
    pages, n = torch.randperm(8, generator=g).view(2, 4).int().to(cuda), torch.tensor([50, 64], dtype=torch.int32, device=cuda)
    kc2, vc2 = kc.clone(), vc.clone()
    a, none = gdn.qk_norm_rope(q, k, at, f, v=v, k_cache=kc, v_cache=vc, rows=rows, output_k=False)
    assert none is None and torch.equal(a, z.qk_norm_rope_cache(q, k, v, at, f, kc2, vc2, rows))
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    assert torch.equal(gdn.window_attn_step(q[0, :2], kc, vc, n, pages=pages), z.window_attn_step(q[0, :2], kc, vc, n, None, 0, None, pages))
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(z.qk_norm_rope.default, (q, k, at, f), test_utils=tests)
    torch.library.opcheck(z.qk_norm_rope_cache.default, (q, k, v, at, f, kc, vc, rows), test_utils=tests)
    torch.library.opcheck(z.window_attn_fwd.default, (q, k, v, 20, 2), test_utils=tests)
    torch.library.opcheck(z.window_attn_step.default, (q[0, :2], kc, vc, n, None, 0, None, pages), test_utils=tests)


@pytest.mark.gpu
def test_host_layer_refuses(gdn, cuda):
    """What the Python layer refuses, with messages, before a launch."""
    bf, f32, i32, i64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
    z = lambda *s, dt=bf: torch.zeros(*s, dtype=dt, device=cuda)  # noqa: E731

    def refused(match, f, *a, **k):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **k)

    rope, fwd, step = gdn.qk_norm_rope, gdn.window_attn_fwd, gdn.window_attn_step
    q, k, at, f = z(8, 4, 64), z(8, 2, 64), z(8, dt=i64), z(32, dt=f32)
    refused("k: expected", rope, q, k[:7], at, f)
    refused("k: expected", rope, q, z(8, 2, 128), at, f)
    refused("as the queries", rope, q, k.float(), at, f)
    refused("head dim", rope, z(8, 4, 96), z(8, 2, 96), at, f)
    refused("positions", rope, q, k, at[:7], f)
    refused("positions", rope, q, k, at.float(), f)
    refused("inv_freq", rope, q, k, at, f.to(bf))
    refused("turns 24", rope, q, k, at, z(12, dt=f32))
    refused("turns 128", rope, q, k, at, z(64, dt=f32))
    refused("q_weight", rope, q, k, at, f, z(63))
    refused("share a dtype", rope, q, k, at, f, z(64), z(64, dt=f32))
    refused("need rows", rope, q, k, at, f, v=k)
    refused("nowhere", rope, q, k, at, f, output_k=False)
    refused("rows", rope, q, k, at, f, k_cache=z(2, 16, 2, 64), rows=at.int())
    refused("go together", rope, q, k, at, f, k_cache=z(2, 16, 2, 64), rows=at, v=k)
    refused("k_cache", rope, q, k, at, f, k_cache=z(2, 16, 3, 64), rows=at)
    refused("one stride", rope, q, k, at, f, k_cache=z(2, 16, 2, 128)[..., :64], rows=at)
    refused("as k_cache", rope, q, k, at, f, k_cache=z(2, 16, 2, 64), rows=at, v=k, v_cache=z(1, 16, 2, 64))
    q, k = z(1, 8, 4, 64), z(1, 8, 2, 64)
    refused("q: expected", fwd, q[0], k[0], k[0])
    refused("k: expected", fwd, q, z(2, 8, 2, 64), k)
    refused("v: expected", fwd, q, k, k[:, :7])
    refused("multiple", fwd, q, z(1, 8, 3, 64), z(1, 8, 3, 64))
    refused("window", fwd, q, k, k, window=0)
    refused("sinks", fwd, q, k, k, sinks=-1)
    refused("needs cu_seqlens", fwd, q, k, k, cu_seqlens_k=[0, 8])
    refused("cu_seqlens_k", fwd, q, k[:, :7], k[:, :7], cu_seqlens=[0, 8])
    refused("ends at", fwd, q, k, k, cu_seqlens=[0, 7])
    refused("decreases", fwd, q, k, k, cu_seqlens=[0, 5, 4, 8])
    refused("entries", fwd, q, k, k, cu_seqlens=[0, 8], cu_seqlens_k=[0, 2, 8])
    refused("int32", fwd, q, k, k, cu_seqlens=z(2, dt=i64))
    refused("B == 1", fwd, z(2, 4, 4, 64), z(2, 4, 2, 64), z(2, 4, 2, 64), cu_seqlens=[0, 4])
    c, n = z(3, 16, 2, 64), z(3, dt=i32)
    q = z(3, 4, 64)
    refused("q: expected", step, q[None], c, c, n)
    refused("k_cache", step, q, c.float(), c, n)
    refused("as k_cache", step, q, c, z(2, 16, 2, 64), n)
    refused("lengths", step, q, c, c, n.long())
    refused("lengths", step, q, c, c, n[:2])
    refused("streams' rows", step, q[:2], c, c, n[:2])
    refused("pages", step, q, c, c, n, pages=z(3, 2, dt=i64))
    refused("pages", step, q, c, c, n, pages=z(2, 2, dt=i32))
    refused("power of two", step, q, z(3, 12, 2, 64), z(3, 12, 2, 64), n, pages=z(3, 2, dt=i32))
    refused("multiple", step, z(3, 3, 64), c, c, n)


@pytest.mark.gpu
def test_no_backward(gdn, cuda):
    """A result of inputs that require a gradient raises in backward."""
    q, k = torch.randn(5, 2, 64, device=cuda, requires_grad=True), torch.randn(5, 2, 64, device=cuda)
    at, f = torch.arange(5, device=cuda), torch.ones(8, device=cuda)
    n = torch.full((5,), 1, dtype=torch.int32, device=cuda)
    for name, o in (("qk_norm_rope", gdn.qk_norm_rope(q, k, at, f)[0]), ("window_attn_fwd", gdn.window_attn_fwd(q[None], k[None], k[None])),
                    ("window_attn_step", gdn.window_attn_step(q, k[:, None], k[:, None], n))):
        with pytest.raises(RuntimeError, match=f"{name}: no backward"):
            o.sum().backward()
    with torch.no_grad():
        assert not gdn.window_attn_fwd(q[None], k[None], k[None]).requires_grad

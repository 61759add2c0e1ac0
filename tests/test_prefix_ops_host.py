"""CPU checks of the query/key norm and the shared-prefix attention: arguments are refused with a
status and a message before any CUDA call, and the workspace is sized by the host alone."""

from __future__ import annotations

import pytest

from conftest import ensure_built

A = 0x10000  # a 16-byte aligned address; the calls below return before anything is read


@pytest.fixture(scope="module")
def lib():
    ensure_built()
    from fcv_b200 import _lib

    return _lib.lib()


def norm(lib, **kw):
    a = dict(qkv=A, dtype=1, N=4, stride=3072, heads=16, kv_heads=16, head_dim=64, qw=A, kw=A, eps=1e-6, cos=A, sin=A,
             rows=128, half=32, inter=1, pos=A, q=A, qs=1024, k=A, ks=1024, v=None, vs=1024, kv_rows=None, limit=4)
    a.update(kw)
    return lib.fcv_qk_norm_rope(a["qkv"], a["dtype"], a["N"], a["stride"], a["heads"], a["kv_heads"], a["head_dim"],
                                a["qw"], a["kw"], a["eps"], a["cos"], a["sin"], a["rows"], a["half"], a["inter"],
                                a["pos"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["kv_rows"], a["limit"],
                                None)


def attend(lib, **kw):
    a = dict(q=A, qs=1024, k=A, ks=2048, v=A, vs=2048, rows=640, pk=A, pks=2048, pv=A, pvs=2048, P=100, dtype=1, cu=A,
             base=A, lens=A, B=4, N=4, heads=16, kv_heads=16, head_dim=64, chunk=1, scale=0.125, out=A, os=1024,
             ws=A, ws_bytes=1 << 30)
    a.update(kw)
    return lib.fcv_shared_prefix_attention(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["rows"], a["pk"],
                                           a["pks"], a["pv"], a["pvs"], a["P"], a["dtype"], a["cu"], a["base"],
                                           a["lens"], a["B"], a["N"], a["heads"], a["kv_heads"], a["head_dim"],
                                           a["chunk"], a["scale"], a["out"], a["os"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=7), -1), (dict(N=-1), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(eps=-1.0), -1),
    (dict(eps=float("nan")), -1), (dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(half=0), -2),
    (dict(half=12), -2), (dict(half=40), -2), (dict(qkv=None), -1), (dict(cos=None), -1), (dict(pos=None), -1),
    (dict(q=None), -1), (dict(k=None), -1), (dict(qkv=A + 8), -1), (dict(cos=A + 4), -1), (dict(qw=A + 4), -1),
    (dict(stride=3073), -1), (dict(qs=1028), -1), (dict(ks=1028), -1), (dict(limit=3), -1), (dict(rows=-1), -1),
])
def test_norm_refuses(lib, bad, status):
    assert norm(lib, **bad) == status
    assert b"fcv_qk_norm_rope" in lib.fcv_last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=2), -1), (dict(B=-1), -1), (dict(N=-1), -1), (dict(P=-1), -1), (dict(rows=-1), -1),
    (dict(chunk=-1), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1),
    (dict(head_dim=32), -2), (dict(head_dim=256), -2), (dict(q=None), -1), (dict(k=None), -1), (dict(pv=None), -1),
    (dict(cu=None), -1), (dict(out=None), -1), (dict(base=None), -1), (dict(lens=None), -1), (dict(q=A + 2), -1),
    (dict(out=A + 8), -1), (dict(qs=1025), -1), (dict(ks=1025), -1), (dict(pvs=1025), -1), (dict(os=1025), -1),
    (dict(ws_bytes=16, P=100000), -1), (dict(scale=0.0), -1), (dict(scale=-0.1), -1),
    (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(ws=None, P=100000), -1), (dict(ws=A + 4, P=100000), -1),
])
def test_attention_refuses(lib, bad, status):
    assert attend(lib, **bad) == status
    assert b"fcv_shared_prefix_attention" in lib.fcv_last_error()


def test_empty_calls_return_before_any_launch(lib):
    assert norm(lib, N=0, qkv=None) == 0
    assert attend(lib, N=0, q=None) == 0
    assert attend(lib, B=0, cu=None) == 0


def test_workspace_is_sized_on_the_host(lib):
    size = lib.fcv_shared_prefix_workspace_bytes
    assert size(0, 4, 16, 16, 64, 100, 6400, 0, 1) == 0
    assert size(4, 0, 16, 16, 64, 100, 6400, 0, 1) == 0
    assert size(4, 4, 16, 3, 64, 100, 6400, 0, 1) == 0
    assert size(4, 4, 16, 16, 64, -1, 6400, 0, 1) == 0
    # at least one part of the prefix and one of the own keys: output, maximum and sum of every head
    assert size(4, 4, 16, 16, 64, 100, 6400, 0, 5) == 0
    assert size(64, 64, 32, 8, 128, 4096, 6400, 0, 0) >= 2 * 64 * 32 * (128 * 4 + 8)


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from fcv_b200 import ops

    x = torch.zeros(2, 3 * 64)
    t = torch.zeros(4, 32)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_norm_rope(x, None, None, t, t, i, 1, 1)
    h = torch.zeros(2, 1, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_prefix_attention(h, h, h, h, h, i)

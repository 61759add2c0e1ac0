"""CPU checks of the query/key norm and the shared-prefix attention: arguments are refused with a
status and a message before any CUDA call, and the workspace is sized by the host alone."""

from __future__ import annotations

import re
import struct

import pytest

from conftest import ROOT, ensure_built

A = 0x10000  # a 16-byte aligned address; the calls below return before anything is read


@pytest.fixture(scope="module")
def lib():
    ensure_built()
    from fcv_b200 import _lib

    return _lib.lib()


def norm(lib, **kw):
    from fcv_b200 import _lib

    a = dict(qkv=A, qw=A, kw=A, cos=A, sin=A, pos=A, q=A, k=A, v=0, kv_rows=0, stride=1536, qs=512, ks=512, vs=512,
             limit=4, dtype=1, N=4, heads=8, kv_heads=8, head_dim=64, rows=128, half=32, inter=1, eps=1e-6)
    a.update(kw)
    return lib.fcv_qk_norm_rope(_lib.QK_NORM.pack(*a.values()), None)


def attention(**kw):
    from fcv_b200 import _lib

    a = dict(q=A, k=A, v=A, pk=A, pv=A, cu=A, base=A, lens=A, out=A, qs=1024, ks=2048, vs=2048, rows=640, pks=2048,
             pvs=2048, os=1024, P=100, dtype=1, B=4, N=4, heads=16, kv_heads=16, head_dim=64, chunk=1, scale=0.125)
    a.update(kw)
    return _lib.PREFIX_ATTENTION.pack(*a.values())


def attend(lib, ws=A, ws_bytes=1 << 40, **kw):
    return lib.fcv_shared_prefix_attention(attention(**kw), ws, ws_bytes, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=7), -1), (dict(N=-1), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(eps=-1.0), -1),
    (dict(eps=float("nan")), -1), (dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(half=0), -2),
    (dict(half=12), -2), (dict(half=40), -2), (dict(qkv=0), -1), (dict(cos=0), -1), (dict(pos=0), -1),
    (dict(q=0), -1), (dict(k=0), -1), (dict(qkv=A + 8), -1), (dict(cos=A + 4), -1), (dict(qw=A + 4), -1),
    (dict(stride=1537), -1), (dict(qs=516), -1), (dict(ks=516), -1), (dict(limit=3), -1), (dict(rows=-1), -1),
])
def test_norm_refuses(lib, bad, status):
    assert norm(lib, **bad) == status
    assert b"fcv_qk_norm_rope" in lib.fcv_last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=2), -1), (dict(B=-1), -1), (dict(N=-1), -1), (dict(P=-1), -1), (dict(rows=-1), -1),
    (dict(chunk=-1), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1),
    (dict(head_dim=32), -2), (dict(head_dim=256), -2), (dict(q=0), -1), (dict(k=0), -1), (dict(pv=0), -1),
    (dict(cu=0), -1), (dict(out=0), -1), (dict(base=0), -1), (dict(lens=0), -1), (dict(q=A + 2), -1),
    (dict(out=A + 8), -1), (dict(qs=1025), -1), (dict(ks=1025), -1), (dict(pvs=1025), -1), (dict(os=1025), -1),
    (dict(ws_bytes=16, P=100000), -1), (dict(scale=0.0), -1), (dict(scale=-0.1), -1),
    (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(ws=None, P=100000), -1), (dict(ws=A + 4, P=100000), -1),
])
def test_attention_refuses(lib, bad, status):
    assert attend(lib, **bad) == status
    assert b"fcv_shared_prefix_attention" in lib.fcv_last_error()


@pytest.mark.parametrize("kw", [
    dict(N=1, B=1, qs=1027, os=1029), dict(rows=1, ks=2049, vs=2051), dict(P=1, pks=2049, pvs=2051),
    dict(rows=0, k=A + 2, v=A + 4, ks=2049), dict(P=0, pk=A + 2, pv=A + 4, pks=2049),
])
def test_single_rows_have_any_stride_and_no_rows_any_address(lib, kw):
    """Such a call passes the check of alignment and stops at the workspace, which is refused last."""
    assert attend(lib, ws=A + 4, dtype=0, **kw) == -1
    assert b"workspace" in lib.fcv_last_error()
    if "rows" not in kw and "P" not in kw:  # the norm: its last check is of the rows of its output
        assert norm(lib, N=1, stride=1537, qs=513, ks=513, limit=0) == -1
        assert b"1 rows into 0" in lib.fcv_last_error()


def test_a_scale_that_overflows_in_log2_units_is_refused(lib):
    """The kernels multiply by scale * log2(e), which has to be finite (2.9e38 * 1.44 > 3.4e38)."""
    assert attend(lib, scale=2.9e38, ws=A + 4) == -1 and b"scale" in lib.fcv_last_error()
    assert attend(lib, scale=2.3e38, ws=A + 4) == -1 and b"workspace" in lib.fcv_last_error()


def test_empty_calls_return_before_any_launch(lib):
    assert lib.fcv_qk_norm_rope(None, None) == -1 and lib.fcv_shared_prefix_attention(None, None, 0, None) == -1
    assert norm(lib, N=0, qkv=0) == 0
    assert attend(lib, N=0, q=0) == 0
    assert attend(lib, B=0, cu=0) == 0


def test_workspace_is_sized_on_the_host(lib):
    size = lambda **kw: lib.fcv_shared_prefix_workspace_bytes(attention(**kw))  # noqa: E731
    assert size(N=0) == 0 and size(B=0) == 0 and size(kv_heads=3) == 0 and size(P=-1) == 0
    assert size(dtype=5) == 0 and size(head_dim=96) == 0 and size(rows=-1) == 0
    assert lib.fcv_shared_prefix_workspace_bytes(None) == 0
    # one part of the prefix and one of the own keys at least: output, maximum and sum of every head
    assert size(N=64, B=64, heads=32, kv_heads=8, head_dim=128, P=4096, dtype=0) >= 2 * 64 * 32 * (128 * 4 + 8)


def test_float32_heads_of_128_are_planned_at_one_block_an_sm(lib):
    """128 sequences of 5 to 8 queries behind 200 keys, 8/1 heads of 128: whole blocks take 60 us and parts
    79; whole blocks need no workspace.  Behind 2000 keys parts are faster."""
    shape = dict(N=851, B=128, heads=8, kv_heads=1, head_dim=128, rows=128 * 128, qs=1024, os=1024, dtype=0)
    assert lib.fcv_shared_prefix_workspace_bytes(attention(P=200, **shape)) == 0
    assert lib.fcv_shared_prefix_workspace_bytes(attention(P=2000, **shape)) > 0


def test_bf16_off_the_tensor_cores_is_planned_by_its_own_steps(lib):
    """130 heads to a key head: 191 queries of one sequence behind 200 keys take 41 us in whole blocks, which
    need no workspace, and 199 in parts; one query behind 8000 keys is cut into parts."""
    shape = dict(heads=130, kv_heads=1, head_dim=64, B=1, qs=8320, os=8320)
    assert lib.fcv_shared_prefix_workspace_bytes(attention(N=191, P=200, rows=1408, **shape)) == 0
    assert lib.fcv_shared_prefix_workspace_bytes(attention(N=1, P=8000, rows=64, **shape)) > 0


@pytest.mark.parametrize("P", [3000, 8000, 16384])
def test_key_tensors_without_rows_leave_every_sm_to_the_prefix(lib, P):
    """The workspace is the parts of the prefix alone: no place for an own part, no stretches of own keys
    that would take a share of the SMs."""
    shape = dict(N=64, B=64, heads=32, kv_heads=8, head_dim=128, P=P, qs=4096, os=4096)
    part = 64 * 32 * (128 * 4 + 8)
    size = lib.fcv_shared_prefix_workspace_bytes(attention(rows=0, **shape))
    assert size > 0 and size % part == 0
    assert lib.fcv_shared_prefix_workspace_bytes(attention(rows=64 * 64, **shape)) % part != 0


@pytest.mark.parametrize("name", ["fcv_qk_norm", "fcv_prefix_attention"])
def test_packed_arguments_have_the_layout_of_the_header(name):
    """The format strings against the structures that the header declares, field by field."""
    from fcv_b200 import _lib

    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), (ROOT / "include" / "fcv_b200.h").read_text(), re.S)
    fmt = ""
    for line in body.group(1).split(";"):
        line = line.strip()
        if line:
            kind = "P" if "*" in line else {"long": "l", "int": "i", "float": "f"}[line.split()[0]]
            fmt += kind * (line.count(",") + 1)
    packed = {"fcv_qk_norm": _lib.QK_NORM, "fcv_prefix_attention": _lib.PREFIX_ATTENTION}[name]
    assert packed.size == struct.calcsize("@" + fmt + "0P")  # padded like the C structure
    assert re.sub(r"(\d+)([A-Za-z])", lambda m: m.group(2) * int(m.group(1)), packed.format[1:]).rstrip("x") == fmt


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

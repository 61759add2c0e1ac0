"""Query/key norm with rotation and shared-prefix attention on the GPU, against 64-bit arithmetic.

Tolerances, by arithmetic.  u = eps / 2 of the type (bf16 2^-8, fp32 2^-24) is one rounding.

* norm: the result r = x_a c - x_b s is rounded once (u |r|); in float32 before that, the sum of D
  squares is off by at most (D / 8 + 8) 2^-24 relative (8 values per thread in order, then a tree),
  half of that reaches rsqrt, and rsqrt, three products and an addition add at most 8 roundings:
  (D / 16 + 12) 2^-24 (|x_a c| + |x_b s|).
* attention: let a = softmax-weighted mean of |v|.  Output rounding u |o|; in bf16, P is rounded
  for the product (2^-8 a) while its sum is not, and one exponential in four may come from a
  polynomial of relative error 1.1e-4 (< 2^-12); a score's float32 error is at most
  (D + 4) 2^-24 scale sum |q k|, which moves P by as much, and P's normalisation by as much again;
  sums over n keys: (n + 64) 2^-24 a, for the product and for the sum.  Exponentials 2^-21.
"""

from __future__ import annotations

import random

import pytest

from conftest import ensure_built

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _lib():
    ensure_built()
    from fcv_b200 import _lib as L

    L.lib()
    yield
    assert ops().device_error() == 0


def ops():
    from fcv_b200 import ops as o

    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------ norm and rotation

def tables(half, rows=4096):
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    th = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv
    return th.cos().float(), th.sin().float()


def norm_ref(x, w, cos, sin, pos, eps, inter):
    """(result, magnitude before the rotation's cancellation) of (n, h, D) heads in 64 bits."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    half = cos.shape[1]
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    i = torch.arange(half, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + half)
    out, mag = y.clone(), y.abs()
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, mag


def check_norm(got, ref, mag):
    D = got.shape[-1]
    tol = U[got.dtype] * ref.abs() * (1 + 2.0 ** -7) + (D / 16 + 12) * 2.0 ** -24 * mag
    bad = ((got.double() - ref).abs() > tol).sum().item()
    assert bad == 0, (bad, (got.double() - ref).abs().max().item())


def norm_inputs(n, H, Hkv, D, half, dtype, seed=0, pad=0):
    g = gen(seed)
    width = (H + 2 * Hkv) * D
    qkv = (torch.randn(n, width + pad, generator=g, device=DEV) * 2).to(dtype)[:, :width]
    qw, kw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    cos, sin = tables(half)
    pos = torch.randint(0, 4096, (n,), generator=g, device=DEV, dtype=torch.int32)
    return qkv, qw, kw, cos, sin, pos


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D,half", [(16, 16, 64, 32), (32, 8, 128, 64), (14, 2, 64, 24), (3, 1, 32, 8),
                                          (5, 5, 256, 128), (1, 1, 128, 8), (7, 7, 32, 16)])
@pytest.mark.parametrize("n", [1, 3, 257])
def test_norm_matches_64_bits(dtype, H, Hkv, D, half, n):
    for inter in (True, False):
        qkv, qw, kw, cos, sin, pos = norm_inputs(n, H, Hkv, D, half, dtype, n + D, pad=16 if n == 3 else 0)
        keep = qkv.clone()
        q, k = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv, interleaved=inter)
        heads = keep.unflatten(1, (H + 2 * Hkv, D))
        rq, rk = (norm_ref(heads[:, sl], w, cos, sin, pos, 1e-6, inter)
                  for sl, w in ((slice(0, H), qw), (slice(H, H + Hkv), kw)))
        check_norm(q, *rq)
        check_norm(k, *rk)
        assert torch.equal(qkv, keep)
        # in place: the same bits in the columns of the rows, values untouched
        q2, k2 = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv, interleaved=inter, inplace=True)
        assert torch.equal(q2, q) and torch.equal(k2, k) and q2.data_ptr() == qkv.data_ptr()
        assert torch.equal(qkv[:, (H + Hkv) * D:], keep[:, (H + Hkv) * D:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_into_cache_rows(dtype):
    n, H, Hkv, D = 70, 8, 2, 64
    qkv, qw, kw, cos, sin, pos = norm_inputs(n, H, Hkv, D, 32, dtype, 5)
    q0, k0 = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv)
    cache = torch.randn(200, 2 * Hkv * D + 8, device=DEV).to(dtype)[:, :2 * Hkv * D]
    before = cache.clone()
    rows = torch.randperm(200, generator=gen(1), device=DEV)[:n].to(torch.int32)
    rows[::7] = -1
    q, same = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv, kv_cache=cache, kv_rows=rows)
    assert same is cache and torch.equal(q, q0)
    expect = before.clone()
    kept = rows >= 0
    expect[rows[kept].long()] = torch.cat((k0.flatten(1), qkv[:, (H + Hkv) * D:]), 1)[kept]
    assert torch.equal(cache, expect)


def test_norm_without_weights_zero_rows_and_empty():
    qkv, _, _, cos, sin, pos = norm_inputs(4, 2, 2, 64, 32, torch.float32, 6)
    qkv[1] = 0
    q, k = ops().qk_norm_rope(qkv, None, None, cos, sin, pos, 2, 2, eps=1e-5)
    ref, mag = norm_ref(qkv.unflatten(1, (6, 64))[:, :2], None, cos, sin, pos, 1e-5, True)
    check_norm(q, ref, mag)
    assert q[1].abs().max() == 0 and k[1].abs().max() == 0
    q, k = ops().qk_norm_rope(qkv[:0], None, None, cos, sin, pos[:0], 2, 2)
    assert q.shape == (0, 2, 64) and k.shape == (0, 2, 64)


def test_norm_reports_rows_out_of_range_and_leaves_them():
    qkv, qw, kw, cos, sin, pos = norm_inputs(6, 2, 2, 64, 32, torch.bfloat16, 7)
    pos[2], pos[3] = 4096, -1
    keep = qkv.clone()
    q, k = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, 2, 2, inplace=True)
    assert ops().device_error() == 601
    assert torch.equal(qkv[2:4], keep[2:4]) and not torch.equal(qkv[1], keep[1])
    pos[2] = pos[3] = 0
    cache = torch.zeros(4, 2 * 2 * 64, dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([0, 1, 4, 3, -1, -1], dtype=torch.int32, device=DEV)
    ops().qk_norm_rope(keep, qw, kw, cos, sin, pos, 2, 2, kv_cache=cache, kv_rows=rows)
    assert ops().device_error() == 602
    assert cache[2].abs().max() == 0 and all(cache[r].abs().max() > 0 for r in (0, 1, 3))


def test_norm_refuses_bad_tensors():
    qkv, qw, kw, cos, sin, pos = norm_inputs(4, 2, 2, 64, 32, torch.bfloat16, 8)
    f = ops().qk_norm_rope
    cache = torch.zeros(8, 256, dtype=torch.bfloat16, device=DEV)
    rows = torch.zeros(4, dtype=torch.int32, device=DEV)
    bad = [
        lambda: f(qkv[:, :-1], qw, kw, cos, sin, pos, 2, 2),
        lambda: f(qkv, qw.bfloat16(), kw, cos, sin, pos, 2, 2),
        lambda: f(qkv, qw[:32], kw, cos, sin, pos, 2, 2),
        lambda: f(qkv, qw, kw, cos, sin[:5], pos, 2, 2),
        lambda: f(qkv, qw, kw, cos.double(), sin.double(), pos, 2, 2),
        lambda: f(qkv, qw, kw, cos, sin, pos.long(), 2, 2),
        lambda: f(qkv, qw, kw, cos, sin, pos[:3], 2, 2),
        lambda: f(qkv, qw, kw, cos, sin, pos.cpu(), 2, 2),
        lambda: f(qkv.t(), qw, kw, cos, sin, pos, 2, 2),
        lambda: f(qkv, qw, kw, cos, sin, pos, 2, 2, kv_cache=cache),
        lambda: f(qkv, qw, kw, cos, sin, pos, 2, 2, kv_rows=rows),
        lambda: f(qkv, qw, kw, cos, sin, pos, 2, 2, kv_cache=cache[:, :128], kv_rows=rows),
        lambda: f(qkv, qw, kw, cos, sin, pos, 2, 2, kv_cache=cache.float(), kv_rows=rows),
        lambda: f(qkv, qw, kw, cos, sin, pos, 2, 2, kv_cache=qkv[:, :256], kv_rows=rows),
        lambda: f(qkv[:1].expand(4, -1), qw, kw, cos, sin, pos, 2, 2, inplace=True),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"case {i} was accepted")
    with pytest.raises(TypeError):
        f(qkv.half(), qw, kw, cos, sin, pos, 2, 2)
    from fcv_b200._lib import FcvError

    with pytest.raises(FcvError):  # rows of 8-byte alignment
        f(torch.zeros(4, 388, dtype=torch.bfloat16, device=DEV)[:, 2:386], qw, kw, cos, sin, pos, 2, 2)
    with pytest.raises(FcvError):  # head_dim 96
        f(torch.zeros(4, 96 * 3, dtype=torch.bfloat16, device=DEV), None, None, cos, sin, pos, 1, 1)


# ------------------------------------------------------------------ attention

def attention_ref(q, k, v, pk, pv, q_lens, base, kv_lens, chunk, scale):
    """(o, softmax mean of |v|, score error bound, keys) per row in 64 bits."""
    N, H, D = q.shape
    Hkv, P = pk.shape[1], pk.shape[0]
    G = H // Hkv
    o = torch.zeros(N, H, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    e = torch.zeros(N, H, 1, dtype=torch.float64, device=q.device)
    row = 0
    for nq, b, nk in zip(q_lens, base, kv_lens):
        if nq == 0:
            continue
        K = torch.cat((pk.double(), k[b:b + nk].double())).repeat_interleave(G, 1).permute(1, 2, 0)
        V = torch.cat((pv.double(), v[b:b + nk].double())).repeat_interleave(G, 1).permute(1, 0, 2)
        Q = q[row:row + nq].double().permute(1, 0, 2) * scale
        key = torch.arange(P + nk, device=q.device)
        seen = torch.ones(nq, P + nk, dtype=torch.bool, device=q.device)
        if chunk > 0:
            at = P + nk - nq + torch.arange(nq, device=q.device)
            seen = torch.div(key, chunk, rounding_mode="floor")[None] <= torch.div(
                at, chunk, rounding_mode="floor")[:, None]
            seen = seen | (key < P)[None]
        if P + nk:
            s = (Q @ K).masked_fill(~seen, float("-inf"))
            m = s.amax(-1, keepdim=True).clamp(min=-1e300)
            p = (s - m).exp()
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            o[row:row + nq] = (p @ V).permute(1, 0, 2)
            a[row:row + nq] = (p @ V.abs()).permute(1, 0, 2)
            e[row:row + nq] = (Q.abs() @ K.abs()).amax(-1).t()[..., None]
        row += nq
    return o, a, e


def check_attention(got, ref, keys):
    o, a, e = ref
    D, u = got.shape[-1], U[got.dtype]
    rel = 2 * (D + 4) * 2.0 ** -24 * e + 2.0 ** -21 + 2 * (keys + 64) * 2.0 ** -24
    if got.dtype == torch.bfloat16:
        rel = rel + 2.0 ** -8 + 2.0 ** -12
    tol = u * (1 + 2.0 ** -7) * (o.abs() + rel * a) + rel * a
    off = (got.double() - o).abs()
    assert torch.isfinite(got).all()
    bad = (off > tol).sum().item()
    assert bad == 0, (bad, off.max().item(), (off / tol.clamp(min=1e-30)).max().item())


def attention_inputs(q_lens, past, P, H, Hkv, D, dtype, seed=0, extra=0, poison=True):
    """past None: own keys are the packed rows; else a cache with capacity behind every sequence, whose
    stale rows hold NaN and infinities."""
    g = gen(seed)
    N, B = sum(q_lens), len(q_lens)
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)) if B else [0], dtype=torch.int32, device=DEV)
    pre = torch.randn(P, 2 * Hkv * D, generator=g, device=DEV).to(dtype)
    pk, pv = (x.unflatten(1, (Hkv, D)) for x in pre.split(Hkv * D, 1))
    if past is None:
        qkv = torch.randn(N + extra, (H + 2 * Hkv) * D, generator=g, device=DEV).to(dtype)
        q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], 1)
        q, k, v = q.unflatten(1, (H, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, D))
        return dict(q=q, k=k, v=v, prefix_k=pk, prefix_v=pv, cu_seqlens=cu), [int(c) for c in cu[:-1]], list(q_lens)
    kv_lens = [a + b for a, b in zip(q_lens, past)]
    cap = max(kv_lens) + 3
    cache = torch.randn(B * cap, 2 * Hkv * D, generator=g, device=DEV).to(dtype)
    base = [b * cap + (b % 3) for b in range(B)]
    if poison:
        used = torch.zeros(B * cap, dtype=torch.bool, device=DEV)
        for b, n in zip(base, kv_lens):
            used[b:b + n] = True
        cache[~used] = float("nan")
        cache[~used, ::3] = float("inf")
    k, v = (x.unflatten(1, (Hkv, D)) for x in cache.split(Hkv * D, 1))
    q = torch.randn(N + extra, H, D, generator=g, device=DEV).to(dtype)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(q=q, k=k, v=v, prefix_k=pk, prefix_v=pv, cu_seqlens=cu, kv_base=t(base), kv_lens=t(kv_lens)), base, \
        kv_lens


def run_case(q_lens, past, P, H, Hkv, D, dtype, chunk, seed=0, scale=None):
    args, base, kv_lens = attention_inputs(q_lens, past, P, H, Hkv, D, dtype, seed)
    got = ops().shared_prefix_attention(**args, chunk=chunk, scale=scale)
    ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], q_lens, base, kv_lens,
                        chunk, D ** -0.5 if scale is None else scale)
    check_attention(got, ref, P + max(kv_lens))
    again = ops().shared_prefix_attention(**args, chunk=chunk, scale=scale)
    assert torch.equal(got, again)
    return got


HEADS = [(16, 16, 64), (14, 2, 64), (8, 2, 128), (3, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("P", [0, 1, 63, 64, 65, 700])
def test_decode_matches_64_bits(dtype, H, Hkv, D, P):
    run_case([1] * 5, [0, 1, 63, 64, 300], P, H, Hkv, D, dtype, 1, P)
    run_case([1], [0], P, H, Hkv, D, dtype, 1, P + 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("chunk", [0, 1, 7, 50])
def test_ragged_queries_match_64_bits(dtype, H, Hkv, D, chunk):
    run_case([1, 0, 130, 37, 64, 5], None, 90, H, Hkv, D, dtype, chunk, chunk)
    run_case([33, 1, 129], [0, 70, 11], 65, H, Hkv, D, dtype, chunk, chunk + 1)
    run_case([2, 3], [0, 0], 0, H, Hkv, D, dtype, chunk, chunk + 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("chunk", [0, 1, 50])
def test_long_queries_match_64_bits(dtype, chunk):
    run_case([700, 383, 1, 512], None, 333, 4, 2, 64, dtype, chunk, 3)
    run_case([385, 640], [0, 129], 128, 2, 2, 128, dtype, chunk, 4)


def test_many_streams_and_long_prefix():
    rng = random.Random(0)
    run_case([1] * 200, [rng.randint(0, 500) for _ in range(200)], 2500, 8, 2, 64, torch.bfloat16, 1, 1)
    run_case([1] * 3, [2000, 0, 17], 9000, 8, 1, 128, torch.bfloat16, 1, 2)
    run_case([3] * 40, [rng.randint(0, 90) for _ in range(40)], 1000, 16, 16, 64, torch.bfloat16, 50, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing_are_zero_and_rows_behind_stay(dtype):
    H, Hkv, D = 4, 2, 64
    # own keys fewer than queries: the first queries stand before every own key and see the prefix only
    for P in (0, 40):
        args, base, _ = attention_inputs([5, 3, 2], [0, 0, 0], P, H, Hkv, D, dtype, 9, extra=4, poison=False)
        args["kv_lens"] = torch.tensor([2, 0, 2], dtype=torch.int32, device=DEV)
        out = torch.full((14, H, D), 7.0, dtype=dtype, device=DEV)
        got = ops().shared_prefix_attention(**args, chunk=1, out=out)
        assert got is out and (out[10:] == 7).all()
        ref = attention_ref(args["q"][:10], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [5, 3, 2], base,
                            [2, 0, 2], 1, D ** -0.5)
        check_attention(got[:10], ref, P + 2)
        if P == 0:
            assert (got[:3] == 0).all() and (got[5:8] == 0).all() and (got[3:5] != 0).any()


def test_strided_views_scale_and_large_scores():
    H, Hkv, D = 4, 4, 64
    args, base, lens = attention_inputs([70, 9], None, 100, H, Hkv, D, torch.bfloat16, 4)
    wide = torch.full((79, 1000), 3.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:, 104:104 + H * D].unflatten(1, (H, D))
    ops().shared_prefix_attention(**args, chunk=1, scale=0.7, out=out)
    ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [70, 9], base, lens, 1, 0.7)
    check_attention(out, ref, 170)
    assert (wide[:, :104] == 3).all() and (wide[:, 104 + H * D:] == 3).all()
    # scores in the hundreds: the running maximum has to be followed
    args["q"] = args["q"] * 40
    got = ops().shared_prefix_attention(**args, chunk=0)
    ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [70, 9], base, lens, 0,
                        D ** -0.5)
    check_attention(got, ref, 170)


def test_keys_past_32_bit_offsets():
    H, Hkv, D, rows = 2, 2, 128, (1 << 31) // 512 + 4096  # the last rows start past 2^31 elements
    cache = torch.empty(rows, 2 * Hkv * D, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(300, 2 * Hkv * D, generator=gen(2), device=DEV).to(torch.bfloat16)
    cache[-300:] = tail
    k, v = (x.unflatten(1, (Hkv, D)) for x in cache.split(Hkv * D, 1))
    q = torch.randn(140, H, D, generator=gen(3), device=DEV).to(torch.bfloat16)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for lens in ([1], [140]):
        got = ops().shared_prefix_attention(q[:lens[0]], k, v, k[:0], v[:0], t([0, lens[0]]), t([rows - 300]),
                                            t([300]))
        ref = attention_ref(q[:lens[0]], k, v, k[:0], v[:0], lens, [rows - 300], [300], 1, D ** -0.5)
        check_attention(got, ref, 300)
        # the same stretch as the shared prefix
        got = ops().shared_prefix_attention(q[:lens[0]], k[:0], v[:0], k[-300:], v[-300:], t([0, lens[0]]), t([0]),
                                            t([0]))
        ref = attention_ref(q[:lens[0]], k, v, k[-300:], v[-300:], lens, [0], [0], 1, D ** -0.5)
        check_attention(got, ref, 300)


def test_bad_rows_are_reported_and_nothing_outside_is_read():
    args, base, lens = attention_inputs([1, 1], [5, 9], 30, 4, 4, 64, torch.bfloat16, 5, poison=False)
    good = ops().shared_prefix_attention(**args)
    rows = args["k"].shape[0]
    for bad in ([0, rows], [0, -4], [0, rows - 3]):
        a = dict(args, kv_base=torch.tensor(bad, dtype=torch.int32, device=DEV))
        got = ops().shared_prefix_attention(**a)
        assert ops().device_error() == 612
        ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [1, 1], [0, 0],
                            [lens[0], 0], 1, 0.125)
        check_attention(got, ref, 40)
    for cu in ([0, 1, 3], [0, 2, 1], [-1, 1, 2]):
        ops().shared_prefix_attention(**dict(args, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV)))
        assert ops().device_error() == 611
    assert torch.equal(ops().shared_prefix_attention(**args), good)


def test_attention_refuses_bad_tensors():
    args, _, _ = attention_inputs([3, 2], [4, 4], 10, 4, 2, 64, torch.bfloat16, 6, poison=False)
    f = ops().shared_prefix_attention
    q, out = args["q"], torch.empty(5, 4, 64, dtype=torch.bfloat16, device=DEV)
    bad = [
        dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q.transpose(1, 2)), dict(q=q[0]),
        dict(k=args["k"][:-1]), dict(k=args["k"].float()), dict(v=args["v"][:, :1]),
        dict(prefix_v=args["prefix_v"][:3]), dict(cu_seqlens=args["cu_seqlens"].long()),
        dict(cu_seqlens=args["cu_seqlens"].cpu()), dict(kv_base=None), dict(kv_lens=args["kv_lens"][:1]),
        dict(chunk=-1), dict(kv_base=None, kv_lens=None, k=args["k"][:4], v=args["v"][:4]), dict(out=out[:4]), dict(out=out.float()), dict(out=q), dict(cu_seqlens=args["cu_seqlens"][:0]),
        dict(out=out[:1].expand(5, -1, -1)),
    ]
    for i, change in enumerate(bad):
        with pytest.raises(ValueError):
            f(**{**args, **change})
            raise AssertionError(f"case {i} was accepted")
    with pytest.raises(TypeError):
        f(**{n: t.half() if t.dtype == torch.bfloat16 else t for n, t in args.items()})
    # nothing to do
    none = f(q[:0], args["k"], args["v"], args["prefix_k"], args["prefix_v"], args["cu_seqlens"][:1])
    assert none.shape == (0, 4, 64)


# (query lengths, keys before them, prefix, H, Hkv, D) and the kernels that a bf16 call launches
WAYS = {
    "whole, few rows": (([1] * 4, [0, 5, 30, 36], 200, 16, 16, 64), 1),
    "whole, 50-row chunks": (([50] * 12, [0] * 12, 150, 16, 16, 64), 1),
    "whole, tensor cores, heads of 64": (([300, 411, 1, 260] * 4, None, 777, 14, 2, 64), 2),
    "whole, tensor cores, heads of 128": (([300, 411, 1, 260] * 4, None, 500, 32, 8, 128), 2),
    "parts, own keys streamed, heads of 64": (([1] * 40, list(range(0, 400, 10)), 6000, 16, 4, 64), 3),
    "parts, own keys streamed, heads of 128": (([1] * 40, list(range(0, 400, 10)), 6000, 32, 8, 128), 3),
    "parts, shared SMs picked on the device": (([1] * 130, [i % 97 for i in range(130)], 16000, 32, 8, 128), 3),
    "parts, several queries streamed": (([2, 3, 1, 0, 4] * 6, [70] * 30, 5000, 16, 4, 64), 3),
    "parts, rows of a sequence in blocks": (([50, 3, 77], [100, 0, 9], 9000, 16, 16, 64), 3),
    "parts, 20 heads to a key head": (([1, 2, 1], [100, 0, 900], 9000, 20, 1, 128), 3),
    "130 heads to a key head": (([1, 5], [40, 0], 700, 130, 1, 64), 2),
}


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("chunk", [1, 0])
def test_every_way_of_cutting(way, chunk):
    from fcv_b200 import _lib

    (q_lens, past, P, H, Hkv, D), launches = WAYS[way]
    count = _lib.lib().fcv_launch_count
    before = count()
    run_case(q_lens, past, P, H, Hkv, D, torch.bfloat16, chunk, 7)
    assert (count() - before) / 2 == launches  # run_case calls twice
    run_case(q_lens[:8], past and past[:8], min(P, 900), H, Hkv, D, torch.float32, chunk, 8)


def test_expanded_rows():
    """Rows of stride 0 (a TMA tensor may not have them): one key repeated is one key."""
    H, Hkv, D = 8, 2, 64
    g = gen(51)
    q = torch.randn(300, H, D, generator=g, device=DEV).bfloat16()
    one = torch.randn(1, Hkv, D, generator=g, device=DEV).bfloat16()
    cu = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops().shared_prefix_attention(q, one[:0], one[:0], one.expand(2000, -1, -1), one.expand(2000, -1, -1), cu,
                                        none, none)
    want = one.repeat_interleave(H // Hkv, 1).expand(300, -1, -1).double()
    assert ((got.double() - want).abs() <= 2 * 2.0 ** -8 * want.abs()).all()
    # one query and one own key, each a row of stride 0, behind a long prefix
    pre = torch.randn(5000, Hkv, D, generator=g, device=DEV).bfloat16()
    row = torch.randn(H, D, generator=g, device=DEV).bfloat16()
    key = torch.randn(Hkv, D, generator=g, device=DEV).bfloat16()
    args = (pre, pre, torch.tensor([0, 1], dtype=torch.int32, device=DEV), none, none + 1)
    got = ops().shared_prefix_attention(row.expand(1, -1, -1), key.expand(1, -1, -1), key.expand(1, -1, -1), *args)
    assert torch.equal(got, ops().shared_prefix_attention(row[None].clone(), key[None].clone(), key[None].clone(), *args))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("q_lens,past,P,D", [([1, 1, 1], [40, 70, 3], 100, 64), ([1, 1, 1], [40, 70, 3], 6000, 128),
                                             ([200, 150, 90], None, 300, 64), ([300, 250, 90], None, 300, 128),
                                             ([40, 33, 20], [0, 70, 3], 6000, 64)])
def test_not_a_number_in_a_key_stays_with_the_rows_that_see_it(value, q_lens, past, P, D):
    for dtype in (torch.bfloat16, torch.float32):
        args, base, lens = attention_inputs(q_lens, past, P, 8, 2, D, dtype, 61, poison=past is not None)
        clean = ops().shared_prefix_attention(**args)
        at = lens[1] - 2  # the last key but one of the second sequence: seen by its last two queries
        args["k"][base[1] + at, 0, 5] = value
        got = ops().shared_prefix_attention(**args)
        rows = torch.arange(sum(q_lens[:1]) + max(0, q_lens[1] - 2), sum(q_lens[:2]), device=DEV)
        if value != value:
            assert torch.isnan(got[rows][:, :4]).all()  # the four query heads of key head 0
        else:  # a score of +inf or -inf by the query's sign: NaN, or the key left out
            plus = args["q"][rows][:, :4, 5] > 0
            assert torch.isnan(got[rows][:, :4][plus]).all() and torch.isfinite(got[rows][:, :4][~plus]).all()
        got[rows, :4] = clean[rows, :4]
        assert torch.equal(got, clean)


def test_agrees_with_ragged_attention_on_whole_documents():
    """A batch whose documents start with the same rows: the rows behind them, computed with the shared
    keys, agree with the packed attention of the whole documents."""
    H, D, P, chunk = 16, 64, 150, 50  # whole chunks, so the mask cuts neither side differently
    q_lens = [50, 100, 37]
    g = gen(12)
    for dtype in (torch.bfloat16, torch.float32):
        pre = torch.randn(P, 3 * H * D, generator=g, device=DEV).to(dtype)
        own = [torch.randn(n, 3 * H * D, generator=g, device=DEV).to(dtype) for n in q_lens]
        rows = torch.cat([torch.cat((pre, o)) for o in own])
        lens = [P + n for n in q_lens]
        cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)
        tiles, nt = ops().attention_tiles(lens, chunk, DEV)
        whole = ops().ragged_attention(rows, cu, tiles, nt, chunk, max(lens))
        packed = torch.cat(own)
        q, k, v = (x.unflatten(1, (H, D)) for x in packed.split(H * D, 1))
        _, pk, pv = (x.unflatten(1, (H, D)) for x in pre.split(H * D, 1))
        cq = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32, device=DEV)
        got = ops().shared_prefix_attention(q, k, v, pk, pv, cq, chunk=chunk)
        at = torch.cat([torch.arange(int(c) + P, int(c) + n) for c, n in zip(cu, lens)]).to(DEV)
        ref = attention_ref(q, k, v, pk, pv, q_lens, [0, 50, 150], q_lens, chunk, 0.125)
        check_attention(got, ref, max(lens))
        check_attention(whole[at].unflatten(1, (H, D)), ref, max(lens))


# ------------------------------------------------------------------ together, streams, graphs

def test_decoding_step_by_step_equals_one_prefill():
    """Projection, norm and rotation into the cache, shared-prefix attention, projection: the tokens of
    three streams run at once and one at a time give the same, within the roundings of bf16."""
    from fcv_b200 import _lib

    o = ops()
    H, Hkv, D, P, T = 16, 4, 64, 130, 9
    g = gen(21)
    dim = 1024
    w = (torch.randn((H + 2 * Hkv) * D, dim, generator=g, device=DEV) / 32).bfloat16()
    wo = (torch.randn(dim, H * D, generator=g, device=DEV) / 32).bfloat16()
    qw, kw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    cos, sin = tables(32)
    x = torch.randn(3 * T, dim, generator=g, device=DEV).bfloat16()
    prompt = torch.randn(P, dim, generator=g, device=DEV).bfloat16()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731

    def layer(rows, pos, cache, kv_rows, cu, base, lens, pk, pv):
        qkv = o.linear(rows, w)
        q, _ = o.qk_norm_rope(qkv, qw, kw, cos, sin, i32(pos), H, Hkv, kv_cache=cache, kv_rows=i32(kv_rows))
        k, v = (t.unflatten(1, (Hkv, D)) for t in cache.split(Hkv * D, 1))
        a = o.shared_prefix_attention(q, k, v, pk, pv, i32(cu), i32(base), i32(lens))
        return o.linear(a.flatten(1), wo, epilogue=_lib.EPI_BIAS_F32)

    pre = torch.zeros(P, 2 * Hkv * D, dtype=torch.bfloat16, device=DEV)
    empty = pre[:0, :Hkv * D].unflatten(1, (Hkv, D))
    layer(prompt, range(P), pre, range(P), [0, P], [0], [P], empty, empty)
    pk, pv = (t.unflatten(1, (Hkv, D)) for t in pre.split(Hkv * D, 1))
    once = torch.zeros(3 * T, 2 * Hkv * D, dtype=torch.bfloat16, device=DEV)
    pos = [P + t for _ in range(3) for t in range(T)]
    whole = layer(x, pos, once, range(3 * T), [0, T, 2 * T, 3 * T], [0, T, 2 * T], [T] * 3, pk, pv)
    steps = torch.zeros_like(once)
    for t in range(T):
        at = [t, T + t, 2 * T + t]
        y = layer(x[at], [P + t] * 3, steps, at, [0, 1, 2, 3], [0, T, 2 * T], [t + 1] * 3, pk, pv)
        # two bf16 attention outputs, each within 2^-8 |o| + 2^-8 a of the exact one, through the same
        # projection of 1024 values: root mean square below 2 * 2^-8 of the output's
        assert (y - whole[at]).norm() <= 2 * 2.0 ** -8 * whole[at].norm()
    assert torch.equal(steps, once)  # a token's cache row does not depend on its company
    # the layer in 64 bits, from the stored keys and values
    q64, _ = norm_ref(o.linear(x, w).unflatten(1, (H + 2 * Hkv, D))[:, :H], qw, cos, sin, i32(pos), 1e-6, True)
    k, v = (t.unflatten(1, (Hkv, D)) for t in once.split(Hkv * D, 1))
    ref, _, _ = attention_ref(q64.bfloat16(), k, v, pk, pv, [T] * 3, [0, T, 2 * T], [T] * 3, 1, 0.125)
    out = ref.flatten(1) @ wo.double().t()
    assert (whole - out).norm() <= 2 * 2.0 ** -8 * out.norm()


def test_side_stream_and_graph_replay_with_new_lengths():
    H, Hkv, D = 8, 2, 64
    o = ops()
    args, base, lens = attention_inputs([1] * 6, [0, 3, 64, 100, 10, 200], 500, H, Hkv, D, torch.bfloat16, 31,
                                        poison=False)
    n = norm_inputs(6, H, Hkv, D, 32, torch.bfloat16, 32)
    cache = torch.zeros(40, 2 * Hkv * D, dtype=torch.bfloat16, device=DEV)
    rows = torch.arange(6, dtype=torch.int32, device=DEV)
    eager = o.shared_prefix_attention(**args)
    eq, _ = o.qk_norm_rope(*n, H, Hkv, kv_cache=cache, kv_rows=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = o.shared_prefix_attention(**args)
            gq, _ = o.qk_norm_rope(*n, H, Hkv, kv_cache=cache, kv_rows=rows)
    side.synchronize()
    assert torch.equal(got, eager) and torch.equal(gq, eq)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = o.shared_prefix_attention(**args)
            z, _ = o.qk_norm_rope(*n, H, Hkv, kv_cache=cache, kv_rows=rows)
        graphs.append(gr)
        outs.append((y, z))
    for gr in graphs + graphs[::-1]:
        gr.replay()
    torch.cuda.synchronize()
    for y, z in outs:
        assert torch.equal(y, eager) and torch.equal(z, eq)
    # lengths are read on the device: a replay follows them
    args["kv_lens"].copy_(torch.tensor([1, 1, 1, 50, 2, 201], dtype=torch.int32))
    graphs[0].replay()
    ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [1] * 6, base,
                        [1, 1, 1, 50, 2, 201], 1, D ** -0.5)
    check_attention(outs[0][0], ref, 701)


def test_replayed_decode_steps_follow_the_lengths():
    """Prefix parts and streamed own keys side by side in a graph: each replay recomputes the cut."""
    o = ops()
    for P, B in ((9000, 24), (16000, 130)):
        args, base, lens = attention_inputs([1] * B, [(37 * b) % 211 for b in range(B)], P, 32, 8, 128, torch.bfloat16, 71)
        o.shared_prefix_attention(**args)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = o.shared_prefix_attention(**args)
        for new in (lens, [1] * B, [max(1, n - 7 * (b % 5)) for b, n in enumerate(lens)], [0] * B):
            args["kv_lens"].copy_(torch.tensor(new, dtype=torch.int32))
            for _ in range(3):
                gr.replay()
            eager = o.shared_prefix_attention(**args)
            assert torch.equal(y, eager)
            ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [1] * B, base, new, 1,
                                128 ** -0.5)
            check_attention(y, ref, P + max(new))


def test_two_calls_at_once_on_two_streams():
    o = ops()
    a, _, _ = attention_inputs([40, 300], None, 700, 8, 2, 128, torch.bfloat16, 41)
    b, _, _ = attention_inputs([1] * 50, [i for i in range(50)], 3000, 8, 2, 128, torch.bfloat16, 42)
    ra, rb = o.shared_prefix_attention(**a), o.shared_prefix_attention(**b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        with torch.cuda.stream(s1):
            got.append((o.shared_prefix_attention(**a), ra))
        with torch.cuda.stream(s2):
            got.append((o.shared_prefix_attention(**b), rb))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


@pytest.mark.parametrize("H,Hkv,D,P", [(32, 8, 128, 8000), (32, 8, 128, 3000), (16, 4, 64, 6000), (20, 1, 128, 9000)])
def test_no_own_keys_at_all_behind_a_long_prefix(H, Hkv, D, P):
    """Key tensors without rows leave the parts of the prefix alone; offsets and lengths that are out of
    range are still reported."""
    from fcv_b200 import _lib

    B = 64
    args, base, _ = attention_inputs([1] * B, [0] * B, P, H, Hkv, D, torch.bfloat16, 91, poison=False)
    args["k"], args["v"] = args["k"][:0], args["v"][:0]
    args["kv_base"].zero_()
    args["kv_lens"].zero_()
    count = _lib.lib().fcv_launch_count
    before = count()
    good = ops().shared_prefix_attention(**args)
    assert count() - before == 2  # the parts of the prefix and their join
    assert ops().device_error() == 0
    ref = attention_ref(args["q"], args["k"], args["v"], args["prefix_k"], args["prefix_v"], [1] * B, [0] * B, [0] * B, 1,
                        D ** -0.5)
    check_attention(good, ref, P)
    lens = args["kv_lens"].clone()
    lens[5] = 3
    assert torch.equal(ops().shared_prefix_attention(**dict(args, kv_lens=lens)), good)
    assert ops().device_error() == 612
    cu = args["cu_seqlens"].clone()
    cu[-1] = B + 2
    got = ops().shared_prefix_attention(**dict(args, cu_seqlens=cu))
    assert ops().device_error() == 611
    assert torch.equal(got[:B - 1], good[:B - 1])
    cu[-1], cu[-2] = B, B - 3
    ops().shared_prefix_attention(**dict(args, cu_seqlens=cu))
    assert ops().device_error() == 611


def way_inputs(way, dtype, extra=4):
    """Inputs of a way of cutting, with the own keys named by offsets, and a sequence without queries at
    the end; `extra` rows of q lie behind the last sequence."""
    (q_lens, past, P, H, Hkv, D), _ = WAYS[way]
    if dtype == torch.float32:
        q_lens, past, P = q_lens[:8], past and past[:8], min(P, 900)
    q_lens, past = q_lens + [0], past and past + [0]
    args, base, kv_lens = attention_inputs(q_lens, past, P, H, Hkv, D, dtype, 81, extra=extra, poison=False)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    args["kv_base"], args["kv_lens"] = t(base), t(kv_lens)
    return args, q_lens, base, kv_lens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("way", list(WAYS))
def test_keys_out_of_range_of_a_sequence_without_queries_are_reported(way, dtype):
    args, q_lens, base, kv_lens = way_inputs(way, dtype)
    good = ops().shared_prefix_attention(**args)
    assert ops().device_error() == 0
    args["kv_base"][-1], args["kv_lens"][-1] = args["k"].shape[0] - 1, 2
    got = ops().shared_prefix_attention(**args)
    assert ops().device_error() == 612
    used = sum(q_lens)
    assert torch.equal(got[:used], good[:used])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("way", list(WAYS))
def test_bad_rows_in_every_way_of_cutting(way, dtype):
    """Own keys out of range cost their sequence its own keys and nothing else; offsets out of order or
    range spare the rows that lie outside the refused pairs; rows behind the last sequence stay."""
    args, q_lens, base, kv_lens = way_inputs(way, dtype)
    P, D, used, N, rows = args["prefix_k"].shape[0], args["q"].shape[2], sum(q_lens), args["q"].shape[0], args["k"].shape[0]
    j = next(b for b in range(1, len(q_lens)) if q_lens[b] > 0 and kv_lens[b] > 1)
    inputs = [args[n] for n in ("q", "k", "v", "prefix_k", "prefix_v")]
    full = [x[:used] for x in attention_ref(*inputs, q_lens, base, kv_lens, 1, D ** -0.5)]
    start = sum(q_lens[:j])
    alone = attention_ref(inputs[0][start:], *inputs[1:], [q_lens[j]], [0], [0], 1, D ** -0.5)
    without = [x.clone() for x in full]
    for x, y in zip(without, alone):
        x[start:start + q_lens[j]] = y[:q_lens[j]]

    def call(error, **change):
        out = torch.full((N,) + tuple(args["q"].shape[1:]), 7.0, dtype=dtype, device=DEV)
        ops().shared_prefix_attention(**{**args, **change}, out=out)
        assert ops().device_error() == error
        return out

    for name, value in (("kv_base", rows), ("kv_base", rows - 1), ("kv_base", -4), ("kv_lens", -5),
                        ("kv_lens", rows + 1)):
        bad = args[name].clone()
        bad[j] = value
        out = call(612, **{name: bad})
        check_attention(out[:used], without, P + max(kv_lens))
        assert (out[used:] == 7).all()
    cu = args["cu_seqlens"]

    def offsets(at, value, spared, behind=True):
        bad = cu.clone()
        bad[at] = value
        out = call(611, cu_seqlens=bad)
        keep = torch.ones(used, dtype=torch.bool, device=DEV)
        keep[spared[0]:spared[1]] = False
        check_attention(out[:used][keep], [x[keep] for x in full], P + max(kv_lens))
        assert not behind or (out[used:] == 7).all()

    offsets(len(q_lens), N + 3, (used, used), behind=False)  # the last sequence leaves the rows
    offsets(0, -1, (0, q_lens[0]))
    low = int(cu[j]) - 1
    offsets(j + 1, low, (low, int(cu[j + 2]) if j + 2 < len(cu) else used))  # an offset that runs back
    out = call(0)
    check_attention(out[:used], full, P + max(kv_lens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("P,H,Hkv", [(1, 4, 2), (1, 130, 1), (5000, 16, 4)])
def test_single_rows_of_odd_strides(dtype, P, H, Hkv):
    """A row cut out of a buffer of odd width: its stride is never used."""
    D = 64
    odd = lambda n, h, seed: torch.randn(2 * (h * D + 3), generator=gen(seed), device=DEV).to(dtype).as_strided(  # noqa: E731
        (n, h, D), (h * D + 3, D, 1))
    q, k, v = odd(1, H, 1), odd(1, Hkv, 2), odd(1, Hkv, 3)
    if P == 1:
        pk, pv = odd(1, Hkv, 4), odd(1, Hkv, 5)
    else:
        pk, pv = (torch.randn(P, Hkv, D, generator=gen(s), device=DEV).to(dtype) for s in (4, 5))
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = odd(1, H, 6)
    got = ops().shared_prefix_attention(q, k, v, pk, pv, t([0, 1]), t([0]), t([1]), out=out)
    assert got is out
    check_attention(got, attention_ref(q, k, v, pk, pv, [1], [0], [1], 1, D ** -0.5), P + 1)
    # the norm of one such row, into a cache of one
    width = (H + 2 * Hkv) * D
    qkv, qw, kw, cos, sin, pos = norm_inputs(1, H, Hkv, D, 32, dtype, 7)
    row = torch.empty(width + 3, dtype=dtype, device=DEV).as_strided((1, width), (width + 3, 1)).copy_(qkv)
    cache = torch.empty(2 * Hkv * D + 3, dtype=dtype, device=DEV).as_strided((1, 2 * Hkv * D), (2 * Hkv * D + 3, 1))
    q0, k0 = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv)
    q1, _ = ops().qk_norm_rope(row, qw, kw, cos, sin, pos, H, Hkv, kv_cache=cache, kv_rows=t([0]))
    assert torch.equal(q1, q0) and torch.equal(cache[:, :Hkv * D], k0.flatten(1))
    assert torch.equal(cache[:, Hkv * D:], qkv[:, (H + Hkv) * D:])
    q2, k2 = ops().qk_norm_rope(row, qw, kw, cos, sin, pos, H, Hkv, inplace=True)
    assert torch.equal(q2, q0) and torch.equal(k2, k0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("way", list(WAYS))
def test_first_offset_behind_the_first_row_and_a_stretch_of_keys_twice(way, dtype):
    """Rows before the first sequence stay as they were, and two sequences may read one stretch of keys."""
    args, q_lens, base, kv_lens = way_inputs(way, dtype)
    used, P, D = sum(q_lens), args["prefix_k"].shape[0], args["q"].shape[2]
    args["cu_seqlens"] += 3
    base[-2], kv_lens[-2] = base[0], kv_lens[0]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    args["kv_base"], args["kv_lens"] = t(base), t(kv_lens)
    out = torch.full(tuple(args["q"].shape), 7.0, dtype=dtype, device=DEV)
    ops().shared_prefix_attention(**args, out=out)
    assert (out[:3] == 7).all() and (out[3 + used:] == 7).all()
    ref = attention_ref(args["q"][3:3 + used], args["k"], args["v"], args["prefix_k"], args["prefix_v"], q_lens, base,
                        kv_lens, 1, D ** -0.5)
    check_attention(out[3:3 + used], ref, P + max(kv_lens))


@pytest.mark.parametrize("B,q_len,P,H,Hkv,D", [(700, 1, 3000, 16, 4, 64), (1500, 70, 50, 14, 2, 64),
                                               (1300, 3, 20, 4, 2, 64)])
def test_more_sequences_than_threads(B, q_len, P, H, Hkv, D):
    """The kernels that go through the sequences with one block take several of them to a thread."""
    rng = random.Random(B)
    q_lens = [rng.randint(max(1, q_len // 2), q_len) for _ in range(B)]
    past = [rng.randint(0, 90) for _ in range(B)]
    run_case(q_lens, past, P, H, Hkv, D, torch.bfloat16, 1, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("inter", [True, False])
def test_norm_in_place_into_a_cache(dtype, inter):
    """In place with a cache: the query columns are rewritten, keys and values go to the cache alone."""
    n, H, Hkv, D = 70, 14, 2, 64
    qkv, qw, kw, cos, sin, pos = norm_inputs(n, H, Hkv, D, 24, dtype, 15, pad=16)
    keep = qkv.clone()
    q0, k0 = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv, interleaved=inter)
    cache = torch.zeros(90, 2 * Hkv * D, dtype=dtype, device=DEV)
    rows = torch.randperm(90, generator=gen(16), device=DEV)[:n].to(torch.int32)
    q, same = ops().qk_norm_rope(qkv, qw, kw, cos, sin, pos, H, Hkv, interleaved=inter, inplace=True, kv_cache=cache,
                                 kv_rows=rows)
    assert same is cache and q.data_ptr() == qkv.data_ptr() and torch.equal(q, q0)
    assert torch.equal(qkv[:, H * D:], keep[:, H * D:])
    assert torch.equal(cache[rows.long()], torch.cat((k0.flatten(1), keep[:, (H + Hkv) * D:]), 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("way", list(WAYS))
def test_rows_whose_every_score_is_minus_infinity_are_zero(way, dtype):
    args, q_lens, base, kv_lens = way_inputs(way, dtype, extra=0)
    args["q"][..., 5] = args["q"][..., 5].abs() + 1
    args["k"][..., 5] = args["prefix_k"][..., 5] = float("-inf")
    assert (ops().shared_prefix_attention(**args) == 0).all()

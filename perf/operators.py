"""Cases of the packed-attention operators, for timing and for comparison with 64-bit arithmetic.

Two operators that stand next to the packed ragged attention of the estimator:

``qk_norm_rope``
    RMS norm of every query and key head and the position rotation in one pass over packed
    [Q | K | V] rows, with the keys and values stored into a K/V cache.
``shared_prefix_attention``
    attention of a ragged batch whose sequences share one prefix of keys and values (the prompt of
    one voice) and have their own keys behind it, under the chunk-causal mask.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at
the end) or, with ``own`` set, through the package's entry points.
"""

from __future__ import annotations

import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "faster-cosyvoice_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from fcv_b200 import ops

    return ops


# ------------------------------------------------------------------ cases

def _attention(name, dtype, heads, kv_heads, head_dim, batch, prefix, q_len, past, chunk):
    case = {"op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "batch": batch, "prefix": prefix, "q_min": q_len[0], "q_max": q_len[1], "past_min": past[0],
            "past_max": past[1], "chunk": chunk}
    return case if name is None else {"name": name, **case}


def _norm(name, dtype, heads, kv_heads, head_dim, rotary, interleaved, rows, cached):
    case = {"op": "qk_norm", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "rotary": rotary, "interleaved": interleaved, "rows": rows, "cached": cached}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # four streams of one voice decode a token each right after a short prompt: latency only
        _attention("decode 4 streams p200", "bf16", 16, 16, 64, 4, 200, (1, 1), (0, 36), 1),
        # a busy decoder with grouped heads: 64 streams, a long prompt, up to about a thousand own tokens
        _attention("decode 64 streams p4096 gqa", "bf16", 32, 8, 128, 64, 4096, (1, 1), (0, 1023), 1),
        # the largest decode step: 256 streams, a very long shared context, own contexts to two thousand
        _attention("decode 256 streams p16384 gqa", "bf16", 32, 8, 128, 256, 16384, (1, 1), (64, 2047), 1),
        # 32 streams of the streaming estimator, one 50-frame chunk each behind a 400-frame prompt
        _attention("stream 32x50 p400 chunk50", "bf16", 16, 16, 64, 32, 400, (50, 50), (0, 150), 50),
        # ragged new turns over an odd prefix, heads in groups of seven
        _attention("prefill ragged p777 gqa7", "bf16", 14, 2, 64, 9, 777, (1, 600), (0, 0), 1),
        # long new turns behind a shared document: the largest prefill
        _attention("prefill 16x1024 p4096 gqa", "bf16", 32, 8, 128, 16, 4096, (700, 1024), (0, 0), 1),
        # the exact-fp32 mode: offline documents behind a shared prompt, no mask
        _attention("offline fp32 8x300 p250", "f32", 16, 16, 64, 8, 250, (150, 600), (0, 0), 0),
        # the exact-fp32 mode, one token of each of 16 streams
        _attention("decode fp32 16 streams p1000", "f32", 16, 4, 64, 16, 1000, (1, 1), (0, 400), 1),
        # one token of one stream into its cache: latency only
        _norm("qk norm 1 token", "bf16", 16, 16, 64, 64, True, 1, True),
        # an ordinary prefill with grouped heads, halves rotated, into a cache
        _norm("qk norm 6577 rows gqa cache", "bf16", 32, 8, 128, 128, False, 6577, True),
        # 16 requests of 3000 frames under guidance
        _norm("qk norm 96000 rows", "bf16", 16, 16, 64, 64, True, 96000, False),
        # the exact-fp32 mode, half of each head rotated
        _norm("qk norm fp32 20914 rows", "f32", 16, 16, 64, 32, True, 20914, False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    heads, kv_heads = rng.choice([(16, 16), (32, 8), (14, 2), (16, 4), (8, 1), (12, 12)])
    head_dim = rng.choice([64, 128])
    if rng.random() < 0.35:
        rows = _log_int(rng, 1, 40000)
        rotary = rng.choice([head_dim, head_dim // 2])
        return _norm(None, dtype, heads, kv_heads, head_dim, rotary, rng.random() < 0.5, rows, rng.random() < 0.5)
    if rng.random() < 0.5:  # decode steps
        batch = _log_int(rng, 1, 200)
        past = _log_int(rng, 1, 1800)
        prefix = _log_int(rng, 16, 12000)
        if dtype == "f32":
            batch, prefix = min(batch, 48), min(prefix, 3001)
        return _attention(None, dtype, heads, kv_heads, head_dim, batch, prefix, (1, 1), (0, past), 1)
    q_max = _log_int(rng, 2, 700)
    batch = max(1, min(24, int(_log_int(rng, 300, 9000) / q_max)))
    prefix = _log_int(rng, 8, 3500)
    if dtype == "f32":
        batch, prefix = min(batch, 6), min(prefix, 900)
    return _attention(None, dtype, heads, kv_heads, head_dim, batch, prefix, (max(1, q_max // 3), q_max),
                      (0, rng.choice([0, 0, 90, 333])), rng.choice([0, 1, 1, 50]))


def _lengths(case):
    """(query rows, own keys) of every sequence; they belong to the case, not to the seed."""
    rng = random.Random("%(batch)d %(prefix)d %(q_max)d %(past_max)d" % case)
    q = [rng.randint(case["q_min"], case["q_max"]) for _ in range(case["batch"])]
    past = [rng.randint(case["past_min"], case["past_max"]) for _ in range(case["batch"])]
    return q, [a + b for a, b in zip(q, past)]


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    st = {"case": case, "heads": H, "kv_heads": Hkv, "head_dim": D}
    if case["op"] == "qk_norm":
        rows, half = case["rows"], case["rotary"] // 2
        st["qkv"] = normal(rows, (H + 2 * Hkv) * D, scale=1.7)
        st["q_weight"] = 1.0 + 0.2 * torch.randn(D, generator=g, device=dev)
        st["k_weight"] = 1.0 + 0.2 * torch.randn(D, generator=g, device=dev)
        positions = 4096
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        theta = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * inv[None, :]
        st["cos"], st["sin"] = theta.cos().float(), theta.sin().float()
        first = torch.randint(0, positions, (1,), generator=g, device=dev)
        st["positions"] = ((first + torch.arange(rows, device=dev)) % positions).to(torch.int32)
        st["eps"] = 1e-6
        if case["cached"]:
            cache_rows = rows + rows // 8 + 5
            st["kv_cache"] = normal(cache_rows, 2 * Hkv * D)
            st["kv_rows"] = torch.randperm(cache_rows, generator=g, device=dev)[:rows].to(torch.int32)
        return st
    q_lens, kv_lens = _lengths(case)
    B, N = case["batch"], sum(q_lens)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    st["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    prefix = normal(case["prefix"], 2 * Hkv * D)
    st["prefix_k"] = prefix[:, :Hkv * D].unflatten(1, (Hkv, D))
    st["prefix_v"] = prefix[:, Hkv * D:].unflatten(1, (Hkv, D))
    if case["past_max"] == 0:  # the own keys are the packed rows themselves
        qkv = normal(N, (H + 2 * Hkv) * D)
        st["q"] = qkv[:, :H * D].unflatten(1, (H, D))
        st["k"] = qkv[:, H * D:(H + Hkv) * D].unflatten(1, (Hkv, D))
        st["v"] = qkv[:, (H + Hkv) * D:].unflatten(1, (Hkv, D))
        st["kv_base"] = st["kv_lens"] = None
        base = cu[:-1]
    else:  # the own keys are rows of a cache, a stretch of equal capacity for every sequence
        cap = (max(kv_lens) + 63) // 64 * 64
        cache = normal(B * cap, 2 * Hkv * D)
        st["q"] = normal(N, H, D)
        st["k"] = cache[:, :Hkv * D].unflatten(1, (Hkv, D))
        st["v"] = cache[:, Hkv * D:].unflatten(1, (Hkv, D))
        base = [b * cap for b in range(B)]
        st["kv_base"] = torch.tensor(base, dtype=torch.int32, device=dev)
        st["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device=dev)
    # index tables of the plain form: padded places of the packed rows and of the own keys
    st["max_q"], st["max_kv"] = max(q_lens), max(kv_lens)
    lens = torch.tensor(q_lens, device=dev)
    st["row_seq"] = torch.repeat_interleave(torch.arange(B, device=dev), lens)
    st["row_pos"] = torch.arange(N, device=dev) - torch.tensor(cu[:-1], device=dev)[st["row_seq"]]
    st["lens"] = lens
    st["own_lens"] = torch.tensor(kv_lens, device=dev)
    st["own_base"] = torch.tensor(base, device=dev)
    return st


# ------------------------------------------------------------------ one pass

def _plain_norm(st):
    case, H, Hkv, D = st["case"], st["heads"], st["kv_heads"], st["head_dim"]
    qkv, half = st["qkv"], case["rotary"] // 2
    n = qkv.shape[0]
    pos = st["positions"].long()
    c, s = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]

    def one(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + st["eps"]) * weight
        r, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat((a * c - b * s, b * c + a * s), -1)
        return torch.cat((r, rest), -1).to(qkv.dtype)

    q = one(qkv[:, :H * D].reshape(n, H, D), st["q_weight"])
    k = one(qkv[:, H * D:(H + Hkv) * D].reshape(n, Hkv, D), st["k_weight"])
    if not case["cached"]:
        return q, k
    st["kv_cache"].index_copy_(0, st["kv_rows"].long(),
                               torch.cat((k.reshape(n, Hkv * D), qkv[:, (H + Hkv) * D:]), 1))
    return q, st["kv_cache"]


def _plain_attention(st):
    case, H, Hkv, D = st["case"], st["heads"], st["kv_heads"], st["head_dim"]
    G, B, mq, mk, P = H // Hkv, case["batch"], st["max_q"], st["max_kv"], case["prefix"]
    dev = st["q"].device
    q = torch.zeros(B, mq, H, D, device=dev)
    q[st["row_seq"], st["row_pos"]] = st["q"].float() * D ** -0.5
    q = q.view(B, mq, Hkv, G, D).permute(2, 0, 1, 3, 4).reshape(Hkv, B * mq * G, D)
    sp = torch.bmm(q, st["prefix_k"].float().permute(1, 2, 0)).view(Hkv, B, mq, G, P)
    at = torch.arange(mk, device=dev)
    rows = (st["own_base"][:, None] + torch.minimum(at[None, :], st["own_lens"][:, None] - 1).clamp(min=0))
    ko, vo = st["k"][rows].float(), st["v"][rows].float()  # (B, mk, Hkv, D)
    so = torch.bmm(q.reshape(Hkv * B, mq * G, D), ko.permute(2, 0, 3, 1).reshape(Hkv * B, D, mk))
    so = so.view(Hkv, B, mq, G, mk)
    limit = st["own_lens"][:, None].expand(B, mq)
    if case["chunk"] > 0:
        at_q = P + (st["own_lens"] - st["lens"])[:, None] + torch.arange(mq, device=dev)[None, :]
        limit = torch.minimum(limit, ((at_q // case["chunk"] + 1) * case["chunk"] - P).clamp(min=0))
    so.masked_fill_((at[None, None, :] >= limit[:, :, None])[None, :, :, None, :], float("-inf"))
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp.sub_(m).exp_()
    so.sub_(m).exp_()
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    out = torch.bmm(sp.reshape(Hkv, B * mq * G, P), st["prefix_v"].float().permute(1, 0, 2)).view(Hkv, B, mq, G, D)
    out += torch.bmm(so.reshape(Hkv * B, mq * G, mk), vo.permute(2, 0, 1, 3).reshape(Hkv * B, mk, D)).view(
        Hkv, B, mq, G, D)
    out = (out / total).permute(1, 2, 0, 3, 4).reshape(B, mq, H, D)
    return out[st["row_seq"], st["row_pos"]].to(st["q"].dtype)


def run(state):
    st = state
    if not own:
        return _plain_norm(st) if st["case"]["op"] == "qk_norm" else _plain_attention(st)
    ops = _ops()
    if st["case"]["op"] == "qk_norm":
        return ops.qk_norm_rope(st["qkv"], st["q_weight"], st["k_weight"], st["cos"], st["sin"], st["positions"],
                                st["heads"], st["kv_heads"], eps=st["eps"], interleaved=st["case"]["interleaved"],
                                kv_cache=st.get("kv_cache"), kv_rows=st.get("kv_rows"))
    return ops.shared_prefix_attention(st["q"], st["k"], st["v"], st["prefix_k"], st["prefix_v"],
                                       st["cu_seqlens"], st["kv_base"], st["kv_lens"], chunk=st["case"]["chunk"])


# ------------------------------------------------------------------ work and 64-bit values

def work(case):
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "qk_norm":
        n = case["rows"]
        values = (H + (2 if case["cached"] else 1) * Hkv) * D
        table = min(n, 4096) * case["rotary"] * 4
        return {"bytes": 2 * n * values * es + table + 4 * n * (2 if case["cached"] else 1) + 8 * D,
                "flops": n * (H + Hkv) * D * 7}
    q_lens, kv_lens = _lengths(case)
    P, chunk = case["prefix"], case["chunk"]
    pairs = keys = 0
    for nq, nk in zip(q_lens, kv_lens):
        most = 0
        for i in range(nq):
            seen = nk if chunk == 0 else max(0, min(nk, ((P + nk - nq + i) // chunk + 1) * chunk - P))
            pairs += P + seen
            most = max(most, seen)
        keys += most
    return {"bytes": es * D * (2 * H * sum(q_lens) + 2 * Hkv * (P + keys)), "flops": 4 * D * H * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "qk_norm":
        x = st["qkv"].double().view(case["rows"], H + 2 * Hkv, D)
        half = case["rotary"] // 2
        angle_c = st["cos"].double().index_select(0, st["positions"].long()).unsqueeze(1)
        angle_s = st["sin"].double().index_select(0, st["positions"].long()).unsqueeze(1)
        w = torch.cat((st["q_weight"].double().expand(H, D), st["k_weight"].double().expand(Hkv, D)))
        y = x[:, :H + Hkv]
        y = y / (y.pow(2).sum(-1, keepdim=True) / D + st["eps"]).sqrt() * w
        first = torch.arange(half, device=x.device)
        first, second = (2 * first, 2 * first + 1) if case["interleaved"] else (first, first + half)
        a, b = y[..., first], y[..., second]
        z = y.clone()
        z[..., first] = a * angle_c - b * angle_s
        z[..., second] = a * angle_s + b * angle_c
        if not case["cached"]:
            return z[:, :H], z[:, H:]
        cache = st["kv_cache"].double()
        cache[st["kv_rows"].long()] = torch.cat((z[:, H:], x[:, H + Hkv:]), 1).flatten(1)
        return z[:, :H], cache
    q_lens, kv_lens = _lengths(case)
    P, chunk, G = case["prefix"], case["chunk"], H // Hkv
    out = torch.empty(sum(q_lens), H, D, dtype=torch.float64, device=st["q"].device)
    base = st["own_base"].tolist()
    row = 0
    pk, pv = st["prefix_k"].double(), st["prefix_v"].double()
    for b, (nq, nk) in enumerate(zip(q_lens, kv_lens)):
        k = torch.cat((pk, st["k"][base[b]:base[b] + nk].double())).permute(1, 0, 2)
        v = torch.cat((pv, st["v"][base[b]:base[b] + nk].double())).permute(1, 0, 2)
        x = st["q"][row:row + nq].double().view(nq, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * nq, D)
        score = (x @ k.transpose(1, 2)).view(Hkv, G, nq, P + nk) / D ** 0.5
        key = torch.arange(P + nk, device=x.device)
        if chunk > 0:
            query = P + nk - nq + torch.arange(nq, device=x.device)
            hidden = (key // chunk)[None, :] > (query // chunk)[:, None]
            score = score.masked_fill(hidden & (key >= P)[None, :], float("-inf"))
        y = torch.softmax(score, -1).view(Hkv, G * nq, P + nk) @ v
        out[row:row + nq] = y.view(Hkv, G, nq, D).permute(2, 0, 1, 3).reshape(nq, H, D)
        row += nq
    return out

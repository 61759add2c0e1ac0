"""Torch-facing wrappers of the C-ABI operators.

Names and argument meaning follow the reference's kernel wrappers
(``faster_cosyvoice/token2wav/flashinfer_kernels.py:327-438``) and its
attention runner (``flashinfer_attention.py``), so a caller of those can switch
to these.  Each wrapper only validates, allocates the output with torch and
passes device pointers plus the current stream to ``libfcv_b200.so``.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Sequence

import torch

from . import _lib
from ._lib import call


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.DTYPE_BF16
    if t.dtype == torch.float32:
        return _lib.DTYPE_F32
    raise TypeError(f"unsupported dtype {t.dtype}")


def _s(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _check_rows(*ts):
    for t in ts:
        if t.device.type != "cuda":
            raise ValueError("tensors must live on a CUDA device")


def mask_lengths(mask: torch.Tensor) -> torch.Tensor:
    """int32 document lengths from a (B, 1, T) right-padded 0/1 mask."""
    B, _, T = mask.shape
    m = mask.contiguous()
    out = torch.empty(B, dtype=torch.int32, device=mask.device)
    call("fcv_mask_lengths", m.data_ptr(), _dt(m), B, T, out.data_ptr(), _s(m))
    return out


def pack_layout(lengths: torch.Tensor, padded_length: int, num_rows: int):
    """Device pack layout from int32 device lengths: (gather int64, document_ids,
    positions, cu_seqlens, gap_rows); ``num_rows`` = sum(lengths)."""
    B = lengths.numel()
    dev = lengths.device
    gather = torch.empty(max(num_rows, 1), dtype=torch.int64, device=dev)
    doc = torch.empty(max(num_rows, 1), dtype=torch.int32, device=dev)
    pos = torch.empty(max(num_rows, 1), dtype=torch.int32, device=dev)
    cu = torch.empty(B + 1, dtype=torch.int32, device=dev)
    gap = torch.empty(num_rows + 30 * (B + 1), dtype=torch.int32, device=dev)
    call("fcv_pack_layout", lengths.data_ptr(), B, int(padded_length), int(num_rows), gather.data_ptr(),
         doc.data_ptr(), pos.data_ptr(), cu.data_ptr(), gap.data_ptr(), _s(lengths))
    return gather[:num_rows], doc[:num_rows], pos[:num_rows], cu, gap


def attention_tiles(lengths: Sequence[int], chunk: int, device) -> tuple[torch.Tensor, int]:
    """Work-list entries (doc, q0) of up to 384 query rows (three 128-row query
    tiles sharing K/V), most expensive first (host-built work list)."""
    lengths = [int(x) for x in lengths]
    cap = max(1, sum((L + 127) // 128 for L in lengths))
    buf = (ctypes.c_int32 * (2 * cap))()
    lens = (ctypes.c_int32 * max(1, len(lengths)))(*lengths)
    n = call("fcv_attn_tiles", ctypes.addressof(lens), len(lengths), int(chunk), ctypes.addressof(buf), cap)
    return torch.tensor(list(buf)[:2 * max(n, 1)], dtype=torch.int32).to(device), n


def layer_norm_modulate_packed(hidden: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor,
                               document_ids: torch.Tensor, modulation_stride: int,
                               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``LN(h) * scale[doc] + shift[doc]`` (``flashinfer_kernels.py:327-348``).
    ``shift``/``scale`` are float32 rows ``modulation_stride`` elements apart."""
    _check_rows(hidden, shift, scale, document_ids)
    N = hidden.shape[0]
    out = torch.empty(N, 1024, dtype=out_dtype or hidden.dtype, device=hidden.device)
    call("fcv_ln_modulate", hidden.data_ptr(), _dt(hidden), shift.data_ptr(), scale.data_ptr(),
         document_ids.data_ptr(), int(modulation_stride), N, out.data_ptr(), _dt(out), _s(hidden))
    return out


def gate_residual_layer_norm_modulate_packed(hidden, gate, residual, shift, scale, document_ids,
                                             modulation_stride: int):
    """``h += gate[doc] * r ; norm = LN(h) * scale[doc] + shift[doc]``
    (``flashinfer_kernels.py:351-378``).  Returns (hidden_out, norm)."""
    _check_rows(hidden, gate, residual, shift, scale, document_ids)
    N = hidden.shape[0]
    h_out = torch.empty_like(hidden)
    norm = torch.empty_like(hidden)
    call("fcv_gate_res_ln_modulate", hidden.data_ptr(), gate.data_ptr(), residual.data_ptr(),
         shift.data_ptr(), scale.data_ptr(), document_ids.data_ptr(), int(modulation_stride), N,
         h_out.data_ptr(), norm.data_ptr(), _dt(hidden), _s(hidden))
    return h_out, norm


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           epilogue: int = _lib.EPI_BIAS, out: torch.Tensor | None = None, aux: torch.Tensor | None = None,
           gate: torch.Tensor | None = None, gate_stride: int = 0, rope_cos: torch.Tensor | None = None,
           rope_sin: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` with a fused epilogue (``F.linear`` call sites
    ``flashinfer_dit.py:490, 500, 512, 535``).  bf16 runs on tcgen05 tensor
    cores, fp32 on CUDA cores.  ``bias``, ``gate`` and RoPE tables are fp32.

    * ``EPI_BIAS_ROPE_QKV``: ``aux`` = int32 positions; partial RoPE on Q/K head 0.
    * ``EPI_BIAS_GATE_RES``: ``out`` is the fp32 residual, updated in place as
      ``out += gate[aux[row]] * (x W^T + b)``; ``aux`` = int32 document ids.
    * ``EPI_BIAS_F32``: fp32 output.
    """
    _check_rows(x, weight)
    M, K = x.shape
    Nout = weight.shape[0]
    if weight.shape[1] != K or weight.dtype != x.dtype:
        raise ValueError("weight must be (Nout, K) with the dtype of x")
    if out is None:
        odt = torch.float32 if epilogue in (_lib.EPI_BIAS_F32, _lib.EPI_BIAS_GATE_RES) else x.dtype
        out = torch.empty(M, Nout, dtype=odt, device=x.device)
    call("fcv_gemm", x.data_ptr(), weight.data_ptr(), None if bias is None else bias.data_ptr(), M, Nout, K,
         _dt(x), int(epilogue), out.data_ptr(), None if aux is None else aux.data_ptr(),
         None if gate is None else gate.data_ptr(), int(gate_stride),
         None if rope_cos is None else rope_cos.data_ptr(), None if rope_sin is None else rope_sin.data_ptr(),
         _s(x))
    return out


def ragged_attention(qkv: torch.Tensor, cu_seqlens: torch.Tensor, tiles: torch.Tensor, n_tiles: int,
                     chunk: int = 0, max_len: int = 0, sched: torch.Tensor | None = None,
                     sched_ctas: int = 0) -> torch.Tensor:
    """Packed ragged attention over (N, 3072) [Q|K|V] rows (replaces
    ``RaggedAttentionRunner.wrapper.run``, ``flashinfer_dit.py:501``); chunk > 0
    applies the chunk-causal streaming mask (``flashinfer_attention.py:16-33``).
    ``sched``/``sched_ctas``: the balanced item schedule of a prepared layout
    (``PackedLayout.attn_sched``/``attn_ctas``); results do not depend on it."""
    _check_rows(qkv, cu_seqlens, tiles)
    N = qkv.shape[0]
    out = torch.empty(N, 1024, dtype=qkv.dtype, device=qkv.device)
    call("fcv_attention", qkv.data_ptr(), _dt(qkv), cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, N,
         int(max_len), int(chunk), tiles.data_ptr(), int(n_tiles), None if sched is None else sched.data_ptr(),
         int(sched_ctas), out.data_ptr(), _s(qkv))
    return out


_NO_SWITCH = contextlib.nullcontext()


def _on(device: int):
    """Makes ``device`` current for a launch (nothing to do when it already is)."""
    return _NO_SWITCH if device == torch.cuda.current_device() else torch.cuda.device(device)


def _raw_stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _int32(name: str, t: torch.Tensor, n: int, dev: int):
    if t.dtype is not torch.int32 or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on cuda:{dev}")


def _head_rows(name: str, t: torch.Tensor, heads: int, head_dim: int, dtype: torch.dtype,
               dev: int) -> tuple[int, int]:
    """Rows and row stride of a (rows, heads, head_dim) tensor whose heads are packed inside a row."""
    shape = t.shape
    if (len(shape) != 3 or shape[1] != heads or shape[2] != head_dim or t.dtype is not dtype
            or t.get_device() != dev):
        raise ValueError(f"{name} must be (rows, {heads}, {head_dim}) of {dtype} on cuda:{dev}")
    row, head, last = t.stride()
    if (last != 1 or (head != head_dim and heads > 1)) and shape[0] > 0:
        raise ValueError(f"the heads of a {name} row must be contiguous")
    return shape[0], row


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two (row-strided) tensors meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    ends = [t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
            for t in (a, b)]
    return a.data_ptr() < ends[1] and b.data_ptr() < ends[0]


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 rope_cos: torch.Tensor, rope_sin: torch.Tensor, positions: torch.Tensor, heads: int, kv_heads: int,
                 *, eps: float = 1e-6, interleaved: bool = True, inplace: bool = False,
                 kv_cache: torch.Tensor | None = None,
                 kv_rows: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head, then the rotation by position, in one pass.

    ``qkv``: (N, (heads + 2 kv_heads) head_dim) packed [Q | K | V] rows (rows may be strided),
    head_dim 32, 64, 128 or 256.  Each query and key head becomes ``x * rsqrt(mean(x^2) + eps) *
    weight`` (float32 ``q_weight`` / ``k_weight`` of head_dim values, None = 1); then its first
    ``2 * rope_cos.shape[1]`` values are rotated by ``rope_cos/rope_sin[positions[n]]`` (float32
    tables, int32 positions) over the pairs (2i, 2i + 1) (``interleaved``, the convention of the
    estimator's tables) or (i, i + half).  Values are not touched.

    Returns ``(q, k)``: (N, heads, head_dim) and (N, kv_heads, head_dim), new tensors or, with
    ``inplace``, views of ``qkv``, whose query and key columns are rewritten.  With ``kv_cache``
    (rows, 2 kv_heads head_dim) of [K | V] and int32 ``kv_rows`` (N) the keys and the values go to
    those cache rows instead and ``(q, kv_cache)`` is returned (with ``inplace`` the query columns of
    ``qkv`` are rewritten, its key and value columns stay); a negative row stores nothing (a padding
    token), and the others must differ from one another.  Forward only: the outputs carry no
    gradient.

    A position outside the tables or a row outside the cache is not accessed: the token (its keys
    and values) stays unwritten and :func:`device_error` reports 601 (602)."""
    shape = qkv.shape
    if len(shape) != 2 or heads < 1 or kv_heads < 1 or shape[1] % (heads + 2 * kv_heads):
        raise ValueError("qkv must be (N, (heads + 2 kv_heads) head_dim)")
    N, width = shape
    D = width // (heads + 2 * kv_heads)
    dev = qkv.get_device()
    if dev < 0:
        raise ValueError("tensors must live on a CUDA device")
    dt = _dt(qkv)
    row, last = qkv.stride()
    if (N > 0 and last != 1) or (N > 1 and row < width):
        raise ValueError("qkv rows must be contiguous and must not overlap")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.dtype is not torch.float32 or w.shape != (D,) or w.get_device() != dev
                              or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 tensor of shape ({D},) on cuda:{dev}")
    table = rope_cos.shape
    if (len(table) != 2 or table != rope_sin.shape or rope_cos.dtype is not torch.float32
            or rope_sin.dtype is not torch.float32 or not rope_cos.is_contiguous() or not rope_sin.is_contiguous()
            or rope_cos.get_device() != dev or rope_sin.get_device() != dev):
        raise ValueError(f"rope_cos and rope_sin must be contiguous float32 tables of one shape on cuda:{dev}")
    _int32("positions", positions, N, dev)
    if (kv_cache is None) != (kv_rows is None):
        raise ValueError("kv_cache and kv_rows go together")
    ptr, es, q_width, k_width = qkv.data_ptr(), qkv.element_size(), heads * D, kv_heads * D
    if inplace:
        q, q_row = qkv.as_strided((N, heads, D), (row, D, 1)), row
    else:
        q, q_row = qkv.new_empty((N, heads, D)), q_width
    v_ptr = rows_ptr = 0
    if kv_cache is not None:
        _int32("kv_rows", kv_rows, N, dev)
        if (kv_cache.dim() != 2 or kv_cache.shape[1] != 2 * k_width or kv_cache.dtype is not qkv.dtype
                or kv_cache.get_device() != dev):
            raise ValueError(f"kv_cache must be (rows, {2 * k_width}) of {qkv.dtype} on cuda:{dev}")
        limit = kv_cache.shape[0]
        k_row, last = kv_cache.stride()
        if (limit > 0 and last != 1) or (limit > 1 and k_row < 2 * k_width):
            raise ValueError("kv_cache rows must be contiguous and must not overlap")
        k_ptr = kv_cache.data_ptr() if limit else ptr  # without rows nothing is stored
        if (N > 0 and limit > 0 and k_ptr < ptr + ((N - 1) * row + width) * es
                and ptr < k_ptr + ((limit - 1) * k_row + 2 * k_width) * es):
            raise ValueError("kv_cache must not share memory with qkv")
        v_ptr, rows_ptr, second = k_ptr + k_width * es, kv_rows.data_ptr(), kv_cache
    elif inplace:
        second = qkv.as_strided((N, kv_heads, D), (row, D, 1), qkv.storage_offset() + q_width)
        k_ptr, k_row, limit = ptr + q_width * es, row, N
    else:
        second = qkv.new_empty((N, kv_heads, D))
        k_ptr, k_row, limit = second.data_ptr(), k_width, N
    args = _lib.QK_NORM.pack(
        ptr, 0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
        rope_cos.data_ptr(), rope_sin.data_ptr(), positions.data_ptr(), q.data_ptr(), k_ptr, v_ptr, rows_ptr, row,
        q_row, k_row, k_row, limit, dt, N, heads, kv_heads, D, table[0], table[1], interleaved, eps)
    with _on(dev):
        call("fcv_qk_norm_rope", args, _raw_stream(dev))
    return q, second


def shared_prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor,
                            prefix_v: torch.Tensor, cu_seqlens: torch.Tensor, kv_base: torch.Tensor | None = None,
                            kv_lens: torch.Tensor | None = None, *, chunk: int = 1, scale: float | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged batch whose sequences share one prefix of keys and values.

    ``q``: (N, heads, head_dim) packed query rows, sequence b at ``cu_seqlens[b] ..
    cu_seqlens[b+1]`` (int32).  ``prefix_k`` / ``prefix_v``: (P, kv_heads, head_dim), seen by every
    query, held once for the whole batch; for long prefixes of many short sequences their products run
    over the stacked rows of the batch, otherwise every sequence goes through them.  ``k`` / ``v``: (rows, kv_heads, head_dim);
    sequence b owns rows ``kv_base[b] .. kv_base[b] + kv_lens[b]`` (int32, a cache stretch that ends
    with the keys of its queries), or, without both, the rows of its queries.  Key head j serves
    query heads ``j * heads / kv_heads ...``.  head_dim is 64 or 128; rows may be strided (column
    views of a [Q | K | V] or [K | V] buffer), heads inside a row are packed.

    ``chunk``: 1 is causal, 0 shows every own key, c > 1 is the streaming mask of
    :func:`ragged_attention` over absolute positions (the prefix occupies positions 0 .. P - 1, the
    queries are the last positions of their sequence).  ``scale`` (positive) defaults to
    head_dim ** -0.5.

    Returns ``out`` (N, heads, head_dim); a query that sees no key, or whose every score is -inf, gives
    zeros, rows of ``out`` before ``cu_seqlens[0]`` and behind ``cu_seqlens[-1]`` are not written.  Row
    numbers are checked on the device: :func:`device_error` 612 for own keys outside ``k`` (the
    sequence is computed without own keys), 611 for ``cu_seqlens`` that decrease or leave 0 .. N (rows
    next to such an entry hold nothing of use); nothing outside the tensors is touched.  The cut of the
    keys into parts depends on the batch, so a sequence's result may differ in the last bits with its
    company; equal calls give equal bits.  Forward only: the output carries no gradient."""
    if q.dim() != 3 or prefix_k.dim() != 3:
        raise ValueError("q must be (N, heads, head_dim), prefix_k (P, kv_heads, head_dim)")
    N, H, D = q.shape
    Hkv, dtype, dev = prefix_k.shape[1], q.dtype, q.get_device()
    if dev < 0:
        raise ValueError("tensors must live on a CUDA device")
    dt = _dt(q)
    if Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"{H} query heads do not share {Hkv} key heads evenly")
    _, q_row = _head_rows("q", q, H, D, dtype, dev)
    rows, k_row = _head_rows("k", k, Hkv, D, dtype, dev)
    v_rows, v_row = _head_rows("v", v, Hkv, D, dtype, dev)
    P, pk_row = _head_rows("prefix_k", prefix_k, Hkv, D, dtype, dev)
    pv_rows, pv_row = _head_rows("prefix_v", prefix_v, Hkv, D, dtype, dev)
    if rows != v_rows or P != pv_rows:
        raise ValueError("keys and values must have the same rows")
    B = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
    if B < 0:
        raise ValueError("cu_seqlens must hold at least one entry")
    _int32("cu_seqlens", cu_seqlens, B + 1, dev)
    base_ptr = lens_ptr = 0
    if kv_base is not None and kv_lens is not None:
        _int32("kv_base", kv_base, B, dev)
        _int32("kv_lens", kv_lens, B, dev)
        base_ptr, lens_ptr = kv_base.data_ptr(), kv_lens.data_ptr()
    elif kv_base is not None or kv_lens is not None:
        raise ValueError("kv_base and kv_lens go together")
    elif rows < N:
        raise ValueError("without kv_base, k and v must have a row for every query")
    if chunk < 0:
        raise ValueError("chunk must not be negative")
    if scale is None:
        scale = D ** -0.5
    if out is None:
        out, out_row = torch.empty_like(q) if q.is_contiguous() else q.new_empty((N, H, D)), H * D
    else:
        out_rows, out_row = _head_rows("out", out, H, D, dtype, dev)
        if out_rows != N or (N > 1 and out_row < H * D):
            raise ValueError("out must be (N, heads, head_dim) rows that do not overlap")
        if any(_overlap(out, t) for t in (q, k, v, prefix_k, prefix_v)):
            raise ValueError("out must not share memory with the inputs")
    args = _lib.PREFIX_ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), cu_seqlens.data_ptr(),
        base_ptr, lens_ptr, out.data_ptr(), q_row, k_row, v_row, rows, pk_row, pv_row, out_row, P, dt, B, N, H, Hkv, D,
        chunk, scale)
    with _on(dev):
        need = _lib.lib().fcv_shared_prefix_workspace_bytes(args)
        # a workspace of this call alone, from the allocator that knows streams and graph captures
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        call("fcv_shared_prefix_attention", args, None if ws is None else ws.data_ptr(), need, _raw_stream(dev))
    return out


def unpack_output(packed: torch.Tensor, cu_seqlens: torch.Tensor, padded_length: int) -> torch.Tensor:
    """(N, 80) packed rows -> zero-padded (B, 80, T) (``flashinfer_dit.py:536-543``)."""
    B = cu_seqlens.numel() - 1
    out = torch.empty(B, 80, padded_length, dtype=packed.dtype, device=packed.device)
    call("fcv_unpack_output", packed.contiguous().data_ptr(), _dt(packed), cu_seqlens.data_ptr(), B,
         int(padded_length), packed.shape[0], out.data_ptr(), _s(packed))
    return out


def cfg_euler_(x: torch.Tensor, d: torch.Tensor, dt: float, cfg_rate: float,
               x_next: torch.Tensor | None = None) -> torch.Tensor:
    """In place ``x += dt * ((1+r) d[:R] - r d[R:])`` on float32 x (``flashinfer_flow.py:66-70``)."""
    R, _, T = x.shape
    call("fcv_cfg_euler", x.data_ptr(), d.data_ptr(), _dt(d), R, T, float(dt), float(cfg_rate),
         None if x_next is None else x_next.data_ptr(),
         _lib.DTYPE_BF16 if x_next is None else _dt(x_next), _s(x))
    return x


def device_error(device=None) -> int:
    """Read and clear the library's device error word (0 = none)."""
    code = ctypes.c_int(0)
    dev = torch.device(device or "cuda")
    call("fcv_device_error", ctypes.byref(code), torch.cuda.current_stream(dev).cuda_stream)
    return code.value

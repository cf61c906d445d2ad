"""Serving: algebraic attention of new tokens over a paged key and value cache on MI355X.

The reference scores and samples by running whole rows (src/algebraic/benchmarking.py:170-190);
here a step takes only the new tokens. One layer's step is

    q = paged_append(q, k, v, k_pages, v_pages, page_table, cu_seqlens, kv_lens,
                     q_gain, k_gain, cos, sin)               # norm, rotation, and into the cache
    o = paged_flash_attention(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, sink, n=n, c=c)

for new tokens packed one sequence after the other (one each, chunks of prompts, or both). The
attention is ``flash_attention``'s (src/algebraic/kernels/flash.py:763-857, ``kind="asinh"``), the
norm and rotation those of src/algebraic/model.py:170-174. bfloat16, hand-written HIP
(csrc/paged_decode.hip, packed_fwd.hip, paged_append.hip), no CPU fallback and no gradient. Neither
call reads device data on the host, so a captured graph of a step serves any lengths.

The cache: ``k_pages``, ``v_pages`` (pages, Hkv, page, D), strides in any order with a contiguous
last axis ((pages, page, Hkv, D) storage is a transposed view), page a multiple of 16, D 64 or 128.
``page_table`` (S, width) int32: position i of sequence s lies in page ``page_table[s, i // page]``;
entries behind a sequence's end are not read, sequences may share pages that are only read.
``cu_seqlens`` (S + 1) int32: sequence s's new tokens are ``cu_seqlens[s]:cu_seqlens[s + 1]``.
``kv_lens`` (S) int32: the keys it holds, the new tokens (its last) among them, as many as its row
of the table reaches (``width page``).
"""

import math
from typing import Optional

import torch

from .. import _lib
from .packed import _BF16, _F32, _WEIGHTS, _check_heads, _check_index, _check_scale, _rows, _sink_vector


def _pages(name, t, Hkv, D, device):
    """Pointer and strides (pages, heads, places) of a cache's pages, as the C entry points take them."""
    if t.dtype is not _BF16:
        raise NotImplementedError(f"dtype {t.dtype}: the gfx950 cache kernels take bfloat16")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    (ps, hs, ts, one), at = t.stride(), t.data_ptr()
    if t.shape[0] == 1:  # an axis of length one: its stride says nothing
        ps = D
    if Hkv == 1:
        hs = D
    if one != 1 or (ps | hs | ts) & 7 or ps < D or ts < D or hs < D or at & 15:
        raise ValueError(f"{name}: the last axis must be contiguous and the others start on 16 bytes")
    return at, ps, hs, ts


def _check_cache(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, Hkv):
    """Checks a cache, its table and lengths; returns (pages, page, S, width, the pages' arguments)."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[1] != Hkv or k_pages.shape[3] != q.shape[2]:
        raise ValueError(f"k_pages and v_pages must share the shape (pages, Hkv, page, {q.shape[2]})")
    pages, _, page, D = k_pages.shape
    dev = q.device
    if D != 128 and D != 64:
        raise NotImplementedError(f"head_dim {D}: the gfx950 cache kernels are built for 64 and 128")
    if pages == 0 or page == 0 or page % 16:
        raise NotImplementedError(f"{pages} pages of {page} positions: pages hold a positive multiple of 16")
    where = _pages("k_pages", k_pages, Hkv, D, dev) + _pages("v_pages", v_pages, Hkv, D, dev)
    if kv_lens.dim() != 1:
        raise ValueError("kv_lens must be (S,)")
    S = kv_lens.shape[0]
    _check_index("kv_lens", kv_lens, (S,), dev)
    _check_index("cu_seqlens", cu_seqlens, (S + 1,), dev)
    if page_table.dim() != 2 or page_table.shape[0] != S or page_table.shape[1] == 0:
        raise ValueError(f"page_table must be ({S}, width)")
    width = page_table.shape[1]
    _check_index("page_table", page_table, (S, width), dev)
    return pages, page, S, width, where


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad() or on detached "
                                          "tensors")


def _gains(q_gain, k_gain, device):
    """Both gains in one of the types that the kernel reads, 16-byte aligned, and its code."""
    if (q_gain is not None and k_gain is not None and q_gain.dtype is k_gain.dtype and q_gain.dtype in _WEIGHTS and
            q_gain.device == device and k_gain.device == device):
        return _lib.aligned16(q_gain), _lib.aligned16(k_gain), _WEIGHTS[q_gain.dtype]
    gains = [None if g is None else g.detach() for g in (q_gain, k_gain)]
    types = {g.dtype for g in gains if g is not None}
    same = types.pop() if len(types) == 1 else _F32
    if same not in _WEIGHTS:
        same = _F32
    for i, g in enumerate(gains):
        if g is not None:
            if g.dtype is not same or g.device != device:
                g = g.to(device=device, dtype=same)
            gains[i] = _lib.aligned16(g)
    return (*gains, _WEIGHTS[same])


def _table(t, device):
    if t is None:
        return None
    if t.dtype is not _F32 or t.device != device or t.requires_grad:
        t = t.detach().to(device=device, dtype=_F32)
    return _lib.aligned16(t)


def paged_append(q, k, v, k_pages, v_pages, page_table, cu_seqlens, kv_lens, q_gain=None, k_gain=None, cos=None,
                 sin=None, *, eps: float = 1e-5):
    """Norm and rotate the new tokens' q (N, H, D) and k (N, Hkv, D) and put k and v into the cache.

    Token t of sequence s stands at position ``kv_lens[s] - new + t``, ``new`` the number of its new
    tokens; q and k become ``rot(x / rms(x) gain)`` in f32, rounded once, with the tables' row of that
    position (``cos``, ``sin`` (>= width page, D/2) float32, or both None: no rotation) and gains (D,)
    or None. Returns the queries (N, H, D); ``k_pages`` and ``v_pages`` are written in place, one
    place a token. A token whose position or page number is out of range is not written; queries at
    such a position, and those behind the last sequence, are zero. A place given to two tokens of a
    call (a page that two sequences write) may end up with parts of both.
    """
    _check_heads(q, k, v)
    (N, H, D), Hkv, dev = q.shape, k.shape[1], q.device
    pages, page, S, width, where = _check_cache(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, Hkv)
    if not (eps > 0) or not math.isfinite(eps):
        raise ValueError("eps must be positive and finite")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin are given together")
    reach, rows = width * page, 0
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dim() != 2 or t.shape[0] < reach or t.shape[1] != D // 2:
                raise ValueError(f"{name} must be (>= {reach}, {D // 2})")
        rows = min(cos.shape[0], sin.shape[0])
    for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
        if g is not None and g.numel() != D:
            raise ValueError(f"{name} must have {D} entries")
    _no_gradient("paged_append", q, k, v, k_pages, v_pages, q_gain, k_gain)
    if not q.is_cuda:
        raise RuntimeError("paged_append needs GPU tensors (no CPU fallback)")
    out = q.new_empty(N, H, D)
    if N == 0 or S == 0:
        return out.zero_()
    (q, q_at), (k, k_at), (v, v_at) = _rows(q), _rows(k), _rows(v)
    page_table, cu, kv = page_table.contiguous(), cu_seqlens.contiguous(), kv_lens.contiguous()
    gq, gk, gain_dtype = _gains(q_gain, k_gain, dev)
    cs, sn = _table(cos, dev), _table(sin, dev)
    p = _lib.ptr
    with _lib.device_of(q):
        _lib.check(_lib.load().alg_paged_append(
            _lib.stream_of(q), N, S, H, Hkv, D, *q_at, *k_at, *v_at, *where, pages, page,
            p(page_table), width, p(cu), p(kv), p(gq), p(gk), gain_dtype, p(cs), p(sn), rows, eps, p(out)),
            "paged_append")
    return out


def paged_flash_attention(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, sink_logit: Optional[torch.Tensor] = None,
                          *, n: int = 16, c: float = 16.0):
    """Attention of the new tokens q (N, H, D) over the keys their sequences hold, (N, H, D).

    Token t of sequence s attends to positions up to ``kv_lens[s] - new + t``; query head h reads key
    head ``h // (H // Hkv)``. q's strides as in ``packed_flash_attention``; ``sink_logit`` broadcasts
    to (H,), and -inf switches a head's off. Tokens behind the last sequence, or before position 0, get
    zeros. What pages hold behind a sequence's end is not read; a page number outside the cache makes
    the outputs that would have read it NaN (and may those of tokens before them in the call). A
    sequence may outgrow its row of the table: tokens at positions from ``width page`` on, which have
    no place in it, get NaN, those before are what they would be. The order of every sum is fixed by
    the shapes, and so is a weight's form in the second product, by the call's average rows (tokens
    times H / Hkv) a sequence: two bfloat16 numbers up to 32 of them, one above.
    """
    if k_pages.dim() != 4:
        raise ValueError("k_pages and v_pages must be (pages, Hkv, page, D)")
    if q.dim() != 3:
        raise ValueError("q must be (tokens, heads, D)")
    if q.dtype is not _BF16:
        raise NotImplementedError(f"dtype {q.dtype}: the gfx950 cache kernels take bfloat16")
    (N, H, D), Hkv, dev = q.shape, k_pages.shape[1], q.device
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"{H} query heads do not share {Hkv} key heads evenly")
    pages, page, S, width, where = _check_cache(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, Hkv)
    _check_scale(n, c)
    sink, sink_dtype, count = _sink_vector(sink_logit, H, dev)
    _no_gradient("paged_flash_attention", q, k_pages, v_pages, sink_logit)
    if not q.is_cuda:
        raise RuntimeError("paged_flash_attention needs GPU tensors (no CPU fallback)")
    o = q.new_empty(N, H, D)
    if N == 0 or S == 0:
        return o.zero_()
    lib = _lib.load()
    q, q_at = _rows(q)
    page_table, cu, kv = page_table.contiguous(), cu_seqlens.contiguous(), kv_lens.contiguous()
    nbytes = lib.alg_paged_attn_workspace_size(N, S, H, Hkv, D, width, page)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    p = _lib.ptr
    with _lib.device_of(q):
        _lib.check(lib.alg_paged_attn(
            _lib.stream_of(q), N, S, H, Hkv, D, *q_at, *where, pages, page, p(page_table), width, p(cu), p(kv),
            p(sink), sink_dtype, count, float(c), int(n), p(o), p(ws), nbytes), "paged_flash_attention")
    return o

"""Serving over a paged cache of 8 bits: half the bytes of ``paged.py``'s, which bound a step's attention.

    q = paged_append_fp8(q, k, v, k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens,
                         q_gain, k_gain, cos, sin)          # norm, rotation, and into the cache
    o = paged_flash_attention_fp8(q, k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens,
                                  sink, n=n, c=c)

are ``paged_append`` and ``paged_flash_attention`` over a cache whose rows (the D values of a token at a
key head) are held as ``e4m3(x 2^-e)`` with one scale ``2^e``, e the least whole number for which
``max |x| 2^-e <= 448``. ``k_pages``, ``v_pages`` (pages, Hkv, page, D) torch.float8_e4m3fn, strides in any
order, multiples of 16, with a contiguous last axis; ``k_scales``, ``v_scales`` (pages, Hkv, page)
torch.float8_e8m0fnu with a contiguous last axis. Everything else (page table, lengths, positions, what is
out of range) is as in ``paged.py``. The stored values are bf16 numbers exactly, so that the attention differs
from that over the stored values by no more than over a bf16 cache; a value differs from what was
put in by 2^-4 of itself, or 2^-18 of its row's largest where that is more. (Values under 2^-126
read as zeros.) A row with an infinity or a NaN is held as NaN: tokens that see it get NaN, others do not.
Hand-written HIP (csrc/paged_decode_fp8.hip, packed_fwd.hip, paged_append.hip), no CPU fallback, no gradient.
"""

import math
from typing import Optional

import torch

from .. import _lib
from .packed import _BF16, _check_heads, _check_index, _check_scale, _rows, _sink_vector
from .paged import _gains, _no_gradient, _table

_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _pages8(name, t, Hkv, D, device):
    """Pointer and strides (pages, heads, places) of pages of bytes, as the C entry points take them."""
    if t.dtype is not _E4M3:
        raise NotImplementedError(f"{name}: dtype {t.dtype}: the 8-bit cache kernels take float8_e4m3fn pages")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    (ps, hs, ts, one), at = t.stride(), t.data_ptr()
    if t.shape[0] == 1:  # an axis of length one: its stride says nothing
        ps = D
    if Hkv == 1:
        hs = D
    if one != 1 or (ps | hs | ts) & 15 or ps < D or ts < D or hs < D or at & 15:
        raise ValueError(f"{name}: the last axis must be contiguous and the others start on 16 bytes")
    return at, ps, hs, ts


def _scales8(name, t, shape, device):
    if t.dtype is not _E8M0:
        raise NotImplementedError(f"{name}: dtype {t.dtype}: the 8-bit cache kernels take float8_e8m0fnu scales")
    if t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} on {device}")
    (ps, hs, one), at, (pages, Hkv, page) = t.stride(), t.data_ptr(), shape
    if pages == 1:
        ps = page
    if Hkv == 1:
        hs = page
    if one != 1 or (ps | hs) & 15 or ps < page or hs < page or at & 15:
        raise ValueError(f"{name}: the last axis must be contiguous and the others start on 16 bytes")
    return at, ps, hs


def _check_cache8(k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens, Hkv, D, dev):
    """Checks a cache, its table and lengths; returns (pages, page, S, width, the pages' arguments)."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[1] != Hkv or k_pages.shape[3] != D:
        raise ValueError(f"k_pages and v_pages must share the shape (pages, Hkv, page, {D})")
    pages, _, page, _ = k_pages.shape
    if D != 128 and D != 64:
        raise NotImplementedError(f"head_dim {D}: the gfx950 cache kernels are built for 64 and 128")
    if pages == 0 or page == 0 or page % 16:
        raise NotImplementedError(f"{pages} pages of {page} positions: pages hold a positive multiple of 16")
    rows = (pages, Hkv, page)
    where = (_pages8("k_pages", k_pages, Hkv, D, dev) + _pages8("v_pages", v_pages, Hkv, D, dev) +
             _scales8("k_scales", k_scales, rows, dev) + _scales8("v_scales", v_scales, rows, dev))
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


def paged_append_fp8(q, k, v, k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens, q_gain=None,
                     k_gain=None, cos=None, sin=None, *, eps: float = 1e-5):
    """``paged_append`` into a cache of 8 bits: the new tokens' q (N, H, D) and k (N, Hkv, D) normed and
    rotated in f64, k rounded (through f32) to 8 bits, v to 8 bits, with a scale a row; returns the queries in bf16.

    Positions, tables, gains, and what is out of range, as in ``paged_append``. Pages and scales are
    written in place, one place a token (two tokens' one place may hold parts of both, a scale of the other's bytes).
    """
    _check_heads(q, k, v)
    (N, H, D), Hkv, dev = q.shape, k.shape[1], q.device
    pages, page, S, width, where = _check_cache8(k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens,
                                                 Hkv, D, dev)
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
    _no_gradient("paged_append_fp8", q, k, v, q_gain, k_gain)
    if not q.is_cuda:
        raise RuntimeError("paged_append_fp8 needs GPU tensors (no CPU fallback)")
    out = q.new_empty(N, H, D)
    if N == 0 or S == 0:
        return out.zero_()
    (q, q_at), (k, k_at), (v, v_at) = _rows(q), _rows(k), _rows(v)
    page_table, cu, kv = page_table.contiguous(), cu_seqlens.contiguous(), kv_lens.contiguous()
    gq, gk, gain_dtype = _gains(q_gain, k_gain, dev)
    cs, sn = _table(cos, dev), _table(sin, dev)
    p = _lib.ptr
    with _lib.device_of(q):
        _lib.check(_lib.load().alg_paged_append_fp8(
            _lib.stream_of(q), N, S, H, Hkv, D, *q_at, *k_at, *v_at, *where, pages, page, p(page_table), width, p(cu),
            p(kv), p(gq), p(gk), gain_dtype, p(cs), p(sn), rows, eps, p(out)), "paged_append_fp8")
    return out


def paged_read_fp8(k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens, *, tokens: int):
    """The keys and values that a cache of 8 bits holds for its sequences' last tokens, (tokens, Hkv, D) bf16 each.

    Sequence s gives its last ``cu_seqlens[s + 1] - cu_seqlens[s]`` positions, packed one sequence after the
    other: what ``paged_append_fp8`` stored with these lengths, or, with ``cu_seqlens`` the running sum of
    ``kv_lens``, all that the sequences hold. The bf16 values are the stored ones exactly. Tokens behind the
    last sequence and before position 0 are zeros; places in no page of the cache NaN.
    """
    if k_pages.dim() != 4:
        raise ValueError("k_pages and v_pages must be (pages, Hkv, page, D)")
    N, Hkv, D, dev = int(tokens), k_pages.shape[1], k_pages.shape[3], k_pages.device
    if N < 0 or Hkv == 0:
        raise ValueError(f"{N} tokens of {Hkv} heads")
    pages, page, S, width, where = _check_cache8(k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens,
                                                 Hkv, D, dev)
    if not k_pages.is_cuda:
        raise RuntimeError("paged_read_fp8 needs GPU tensors (no CPU fallback)")
    k, v = (torch.empty(N, Hkv, D, dtype=_BF16, device=dev) for _ in range(2))
    if N == 0 or S == 0:
        return k.zero_(), v.zero_()
    page_table, cu, kv = page_table.contiguous(), cu_seqlens.contiguous(), kv_lens.contiguous()
    p = _lib.ptr
    with _lib.device_of(k):
        _lib.check(_lib.load().alg_paged_read_fp8(
            _lib.stream_of(k), N, S, Hkv, D, *where, pages, page, p(page_table), width, p(cu), p(kv), p(k), p(v)),
            "paged_read_fp8")
    return k, v


def paged_flash_attention_fp8(q, k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens,
                              sink_logit: Optional[torch.Tensor] = None, *, n: int = 16, c: float = 16.0):
    """``paged_flash_attention`` of the new tokens q (N, H, D) bf16 over a cache of 8 bits, (N, H, D) bf16.

    The values attended to are the stored ones; sinks, positions, zeros and NaN as in
    ``paged_flash_attention``. The order of every sum is fixed by the shapes, and so is a weight's form in the second
    product, as there: two bfloat16 numbers for up to 32 rows a sequence on average, one above.
    """
    if k_pages.dim() != 4:
        raise ValueError("k_pages and v_pages must be (pages, Hkv, page, D)")
    if q.dim() != 3:
        raise ValueError("q must be (tokens, heads, D)")
    if q.dtype is not _BF16:
        raise NotImplementedError(f"dtype {q.dtype}: the gfx950 cache kernels take bfloat16 queries")
    (N, H, D), Hkv, dev = q.shape, k_pages.shape[1], q.device
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"{H} query heads do not share {Hkv} key heads evenly")
    pages, page, S, width, where = _check_cache8(k_pages, v_pages, k_scales, v_scales, page_table, cu_seqlens, kv_lens,
                                                 Hkv, D, dev)
    _check_scale(n, c)
    sink, sink_dtype, count = _sink_vector(sink_logit, H, dev)
    _no_gradient("paged_flash_attention_fp8", q, sink_logit)
    if not q.is_cuda:
        raise RuntimeError("paged_flash_attention_fp8 needs GPU tensors (no CPU fallback)")
    o = q.new_empty(N, H, D)
    if N == 0 or S == 0:
        return o.zero_()
    lib = _lib.load()
    q, q_at = _rows(q)
    page_table, cu, kv = page_table.contiguous(), cu_seqlens.contiguous(), kv_lens.contiguous()
    nbytes = lib.alg_paged_attn_fp8_workspace_size(N, S, H, Hkv, D, width, page)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    p = _lib.ptr
    with _lib.device_of(q):
        _lib.check(lib.alg_paged_attn_fp8(
            _lib.stream_of(q), N, S, H, Hkv, D, *q_at, *where, pages, page, p(page_table), width, p(cu), p(kv),
            p(sink), sink_dtype, count, float(c), int(n), p(o), p(ws), nbytes), "paged_flash_attention_fp8")
    return o

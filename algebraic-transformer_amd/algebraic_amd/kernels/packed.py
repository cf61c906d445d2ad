"""Causal algebraic attention over packed sequences with grouped heads on MI355X.

The reference trains on rows of one length with a key head for every query head
(src/algebraic/model.py:167-181). ``packed_flash_attention`` computes the same attention
(src/algebraic/kernels/flash.py:763-857, ``kind="asinh"`` with the range guard's exactness) for
sequences of different lengths laid one after the other, without padding, and for H query heads
that share Hkv key and value heads in groups; differentiable in q, k, v and the sink. bfloat16;
the arithmetic is hand-written HIP (csrc/packed_fwd.hip, packed_bwd.hip), there is no CPU fallback.
"""

import math

import torch

from .. import _lib
from .autograd import first_order
from .flash import _BUILT_D


_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _rows(t):
    """(tokens, heads, D) with a contiguous last axis, strides of whole 16-byte chunks and rows that
    do not overlap, as the kernels read it (a view of anything else is copied); with its pointer and
    strides (tokens, heads), as the C entry points take them. The stride of an axis of length one
    says nothing, and contiguous() keeps it: D stands in its place."""
    tokens, heads, D = t.shape
    for copied in (False, True):
        ts, hs, one = t.stride()
        if heads == 1:
            hs = D
        if tokens == 1:
            ts = D
        at = t.data_ptr()
        if copied or (one == 1 and not (ts | hs) & 7 and ts >= D and hs >= D and not at & 15 and
                      66 * ts + heads * hs + D < 1 << 30):
            return t, (at, ts, hs)
        t = _lib.aligned16(t)


def _check_scale(n, c):
    if n < 2 or n & (n - 1):
        raise ValueError("asinh kernel needs n to be a power of two")
    if not math.isfinite(c) or c <= 0:
        raise ValueError("asinh scale c must be positive and finite")


def _check_index(name, t, shape, device):
    if t.dtype is not _I32 or t.shape != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")


def _check_heads(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"{name} must be (tokens, heads, D)")
        if t.dtype is not _BF16:
            raise NotImplementedError(f"dtype {t.dtype}: the gfx950 packed kernels take bfloat16")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one device")
    (N, H, D), (Nk, Hkv, Dk) = q.shape, k.shape
    if v.shape != k.shape or Nk != N or Dk != D:
        raise ValueError("q (N, H, D) with k and v (N, Hkv, D)")
    if Hkv == 0 or H == 0 or H % Hkv:
        raise ValueError(f"{H} query heads do not share {Hkv} key heads evenly")


def _sink_vector(sink_logit, H, device):
    """The sink logits, (1,) or (H,), f32 or bf16, on ``device``, with their type's code and number;
    (None, 0, 0) without."""
    if sink_logit is None:
        return None, 0, 0
    count = sink_logit.numel()
    if count != H and count != 1:
        raise ValueError(f"sink_logit must broadcast to ({H},)")
    s = sink_logit
    if s.dtype not in _WEIGHTS or s.device != device:
        s = s.detach().to(device=device, dtype=_F32)
    return s if s.is_contiguous() else s.detach().contiguous(), _WEIGHTS[s.dtype], count


_WEIGHTS = {_BF16: _lib.DTYPE_BF16, _F32: _lib.DTYPE_F32}


class _PackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, sink_logit, sink, n, c):
        lib = _lib.load()
        N, H, D = q.shape
        Hkv, S = k.shape[1], cu.shape[0] - 1
        (q, q_at), (k, k_at), (v, v_at), cu = _rows(q), _rows(k), _rows(v), cu.contiguous()
        sink, sink_dtype, count = sink
        dev = q.device
        o = q.new_empty(N, H, D)
        # The statistic's sign says how a row was computed: its bits are kept as whole numbers, which
        # a hook that stores saved floating tensors in fewer bits leaves as they are.
        stat = torch.empty(N * H, dtype=_I32, device=dev)
        nbytes = lib.alg_packed_attn_fwd_workspace_size(N, S, H, Hkv, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        p = _lib.ptr
        with _lib.device_of(q):
            _lib.check(lib.alg_packed_attn_fwd(
                _lib.stream_of(q), N, S, H, Hkv, D, *q_at, *k_at, *v_at, p(cu), p(sink), sink_dtype,
                count, c, n, p(o), p(stat), p(ws), nbytes), "packed_flash_attention forward")
        ctx.save_for_backward(q, k, v, cu, sink, o, stat)
        ctx.scale = (n, c)
        ctx.sink_meta = None if sink_logit is None else (sink_logit.shape, sink_logit.dtype, sink_logit.device)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, cu, sink, o, stat = ctx.saved_tensors
        lib = _lib.load()
        n, c = ctx.scale
        N, H, D = q.shape
        Hkv, S = k.shape[1], cu.shape[0] - 1
        if do.dtype is not _BF16:
            do = do.to(_BF16)
        (q, q_at), (k, k_at), (v, v_at), (do, do_at) = _rows(q), _rows(k), _rows(v), _rows(do)
        dev = q.device
        dq, dk, dv = q.new_empty(N, H, D), q.new_empty(N, Hkv, D), q.new_empty(N, Hkv, D)
        wants_sink = ctx.sink_meta is not None and ctx.needs_input_grad[4]
        sink_dtype, dsink = 1, None
        if sink is not None:
            sink_dtype = _WEIGHTS[sink.dtype]
        if wants_sink:  # per head in the sink's own type; a shared sink's are added up in f32
            shape, dtype, where = ctx.sink_meta
            dsink = torch.empty(H, dtype=dtype if dtype in _WEIGHTS and sink.numel() == H else _F32, device=dev)
        nbytes = lib.alg_packed_attn_bwd_workspace_size(N, S, H, Hkv, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p = _lib.ptr
        with _lib.device_of(q):
            _lib.check(lib.alg_packed_attn_bwd(
                _lib.stream_of(q), N, S, H, Hkv, D, *q_at, *k_at, *v_at, p(cu), p(sink), sink_dtype,
                0 if sink is None else sink.numel(), c, n, p(o), p(stat), *do_at, p(dq), p(dk), p(dv), p(dsink),
                1 if dsink is None else _WEIGHTS[dsink.dtype], p(ws), nbytes), "packed_flash_attention backward")
        if wants_sink:
            if sink.numel() != H:
                dsink = dsink.sum()
            dsink = dsink.reshape(shape)
            if dsink.dtype is not dtype or where != dev:
                dsink = dsink.to(device=where, dtype=dtype)
        dq, dk, dv, dsink = first_order("packed_flash_attention", o, dq, dk, dv, dsink)
        return dq, dk, dv, None, dsink, None, None, None


def packed_flash_attention(q, k, v, cu_seqlens, sink_logit=None, *, n: int = 16, c: float = 16.0):
    """Causal attention within each of the sequences packed into q (N, H, D), k and v (N, Hkv, D).

    Sequence s is the tokens ``cu_seqlens[s]:cu_seqlens[s + 1]`` (int32, on the device, not
    decreasing, from 0, at most N; sequences may be empty). Tokens behind the last sequence get
    zeros, and zero gradients, so that a captured graph of N tokens serves any lengths. Query head h
    attends over key head ``h // (H // Hkv)``. bfloat16, D up to 128; any strides with a contiguous
    last axis (slices of one projection) are read in place where heads and tokens start on 16 bytes.
    ``sink_logit`` broadcasts to (H,). Returns (N, H, D). Scores may have any size, as
    in ``flash_attention(..., kind="asinh", range_guard=True)``: a weight is right to f32 rounding, or to
    2^-19 of the row's mean weight where that is more. A value that is not finite reaches the outputs
    of its own sequence only. Differentiable once: differentiating the gradients raises.
    """
    _check_heads(q, k, v)
    _check_scale(n, c)
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must hold the sequences' starts and the last one's end")
    _check_index("cu_seqlens", cu_seqlens, cu_seqlens.shape, q.device)
    N, H, D = q.shape
    sink = _sink_vector(sink_logit, H, q.device)
    if D > 128 or D == 0:
        raise NotImplementedError(f"head_dim {D}: gfx950 kernels are built for head_dim <= 128")
    if not q.is_cuda:
        raise RuntimeError("packed_flash_attention needs GPU tensors (no CPU fallback)")
    if N == 0:  # nothing to launch, and gradients of zeros
        o = q + (k.sum() + v.sum())
        return o if sink_logit is None else o + (0 * sink_logit.sum()).to(q.dtype)
    if D in _BUILT_D:
        return _PackedFn.apply(q, k, v, cu_seqlens, sink_logit, sink, int(n), float(c))
    # Zero columns up to the next built width leave the scores as they are; the scale sees the
    # logical width, and the sink is scaled with it (as flash_attention does).
    Dp = next(w for w in _BUILT_D if w >= D)
    grow = math.sqrt(D / Dp)
    pad = lambda t: torch.nn.functional.pad(t, (0, Dp - D))  # noqa: E731
    wide = None if sink_logit is None else sink_logit.float() * grow
    return _PackedFn.apply(pad(q), pad(k), pad(v), cu_seqlens, wide, _sink_vector(wide, H, q.device), int(n),
                           float(c) * grow)[..., :D].contiguous()

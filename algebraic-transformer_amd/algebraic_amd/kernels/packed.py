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
from .flash import _BUILT_D, _sink_gradient, _sink_input, make_variant


def _rows(t):
    """(tokens, heads, D) with a contiguous last axis, strides of whole 16-byte chunks and rows that
    do not overlap, as the kernels read it; a view of anything else is copied."""
    ts, hs, one = t.stride()
    D = t.shape[2]
    if (one == 1 and ts % 8 == 0 and hs % 8 == 0 and ts >= D and (hs >= D or t.shape[1] == 1) and
            t.data_ptr() % 16 == 0 and 66 * ts + t.shape[1] * hs + D < 1 << 30):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strided(t):
    """Pointer and strides (tokens, heads) of a rows tensor, as the C entry points take them."""
    return t.data_ptr(), t.stride(0), max(t.stride(1), t.shape[2])


def _check_scale(n, c):
    make_variant("asinh", n, c)  # n a power of two, c positive and finite


def _check_index(name, t, shape, like):
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {shape}")
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")


def _check_heads(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"{name} must be (tokens, heads, D)")
        if t.dtype != torch.bfloat16:
            raise NotImplementedError(f"dtype {t.dtype}: the gfx950 packed kernels take bfloat16")
        if t.device != q.device:
            raise ValueError("q, k and v must be on one device")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("q (N, H, D) with k and v (N, Hkv, D)")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads do not share {k.shape[1]} key heads evenly")


def _check_sink(sink_logit, q):
    if sink_logit is not None and sink_logit.numel() not in (1, q.shape[1]):
        raise ValueError(f"sink_logit must broadcast to ({q.shape[1]},)")


class _PackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, sink_logit, n, c):
        lib = _lib.load()
        N, H, D = q.shape
        Hkv, S = k.shape[1], cu.shape[0] - 1
        q, k, v, cu = _rows(q), _rows(k), _rows(v), cu.contiguous()
        sink = _sink_input(sink_logit, H, q.device)
        o = torch.empty((N, H, D), dtype=q.dtype, device=q.device)
        # The statistic's sign says how a row was computed: its bits are kept as whole numbers, which
        # a hook that stores saved floating tensors in fewer bits leaves as they are.
        stat = torch.empty(N * H, dtype=torch.int32, device=q.device)
        p = _lib.ptr
        with _lib.device_of(q):
            _lib.check(lib.alg_packed_attn_fwd(
                _lib.stream_of(q), N, S, H, Hkv, D, *_strided(q), *_strided(k), *_strided(v), p(cu), p(sink),
                0 if sink is None else sink.numel(), c, n, p(o), p(stat)), "packed_flash_attention forward")
        ctx.save_for_backward(q, k, v, cu, sink, o, stat)
        ctx.scale = (n, c)
        ctx.sink_meta = None if sink_logit is None else (tuple(sink_logit.shape), sink_logit.dtype)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, cu, sink, o, stat = ctx.saved_tensors
        lib = _lib.load()
        n, c = ctx.scale
        N, H, D = q.shape
        Hkv, S = k.shape[1], cu.shape[0] - 1
        do = _rows(do.to(q.dtype))
        new = lambda *shape: torch.empty(shape, dtype=q.dtype, device=q.device)  # noqa: E731
        dq, dk, dv = new(N, H, D), new(N, Hkv, D), new(N, Hkv, D)
        wants_sink = ctx.sink_meta is not None and ctx.needs_input_grad[4]
        dsink = torch.empty(H, dtype=torch.float32, device=q.device) if wants_sink else None
        nbytes = lib.alg_packed_attn_bwd_workspace_size(N, S, H, Hkv)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        p = _lib.ptr
        with _lib.device_of(q):
            _lib.check(lib.alg_packed_attn_bwd(
                _lib.stream_of(q), N, S, H, Hkv, D, *_strided(q), *_strided(k), *_strided(v), p(cu), p(sink),
                0 if sink is None else sink.numel(), c, n, p(o), p(stat), *_strided(do), p(dq), p(dk), p(dv),
                p(dsink), p(ws), nbytes), "packed_flash_attention backward")
        return dq, dk, dv, None, _sink_gradient(dsink, *ctx.sink_meta) if wants_sink else None, None, None


def packed_flash_attention(q, k, v, cu_seqlens, sink_logit=None, *, n: int = 16, c: float = 16.0):
    """Causal attention within each of the sequences packed into q (N, H, D), k and v (N, Hkv, D).

    Sequence s is the tokens ``cu_seqlens[s]:cu_seqlens[s + 1]`` (int32, on the device, not
    decreasing, from 0, at most N; sequences may be empty). Tokens behind the last sequence get
    zeros, and zero gradients, so that a captured graph of N tokens serves any lengths. Query head h
    attends over key head ``h // (H // Hkv)``. bfloat16, D up to 128; any strides with a contiguous
    last axis (slices of one projection) are read in place where heads and tokens start on 16 bytes.
    ``sink_logit`` broadcasts to (H,). Returns (N, H, D). The weights are exact for scores of any
    size, as ``flash_attention(..., kind="asinh", range_guard=True)``'s are; a value that is not
    finite reaches the outputs of its own sequence only.
    """
    _check_heads(q, k, v)
    _check_scale(n, c)
    _check_sink(sink_logit, q)
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must hold the sequences' starts and the last one's end")
    _check_index("cu_seqlens", cu_seqlens, tuple(cu_seqlens.shape), q)
    D = q.shape[2]
    if D > 128 or D == 0:
        raise NotImplementedError(f"head_dim {D}: gfx950 kernels are built for head_dim <= 128")
    if not q.is_cuda:
        raise RuntimeError("packed_flash_attention needs GPU tensors (no CPU fallback)")
    if q.shape[0] == 0:  # nothing to launch, and gradients of zeros
        o = q + (k.sum() + v.sum())
        return o if sink_logit is None else o + (0 * sink_logit.sum()).to(q.dtype)
    if D in _BUILT_D:
        return _PackedFn.apply(q, k, v, cu_seqlens, sink_logit, int(n), float(c))
    # Zero columns up to the next built width leave the scores as they are; the scale sees the
    # logical width, and the sink is scaled with it (as flash_attention does).
    Dp = next(w for w in _BUILT_D if w >= D)
    grow = math.sqrt(D / Dp)
    pad = lambda t: torch.nn.functional.pad(t, (0, Dp - D))  # noqa: E731
    sink = None if sink_logit is None else sink_logit.float() * grow
    return _PackedFn.apply(pad(q), pad(k), pad(v), cu_seqlens, sink, int(n), float(c) * grow)[..., :D].contiguous()

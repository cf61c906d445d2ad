"""The token embedding on MI355X: the lookup of the table that ``fused_head`` and ``head_logits`` read as the
head's weights (src/algebraic/model.py), and its gradient.

Hand-written HIP (csrc/embedding.hip), no CPU fallback. Neither direction reads device data on the host.
"""

import math
from typing import Optional

import torch

from .. import _lib
from .autograd import first_order

_FLOATS = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_INTS = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, embed, scale, dtype):
        V, d = embed.shape
        tokens, table = tokens.contiguous(), _lib.aligned16(embed)
        N, dev = tokens.numel(), embed.device
        y = torch.empty((*tokens.shape, d), dtype=dtype, device=dev)
        p = _lib.ptr
        with _lib.device_of(embed):
            _lib.check(_lib.load().alg_embedding_fwd(
                _lib.stream_of(embed), N, d, V, p(tokens), _INTS[tokens.dtype], p(table), _FLOATS[table.dtype], scale,
                p(y), _FLOATS[dtype]), "token_embedding")
        ctx.save_for_backward(tokens)
        ctx.meta = (V, d, scale, embed.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        tokens, = ctx.saved_tensors
        V, d, scale, dtype = ctx.meta
        lib = _lib.load()
        cotangent = dy  # all that the gradient depends on: differentiating it by that raises
        dy = _lib.aligned16(dy if dy.dtype in _FLOATS else dy.float())
        N = tokens.numel()
        grad = torch.empty(V, d, dtype=dtype, device=dy.device)
        nbytes = lib.alg_embedding_bwd_workspace_size(N, d, V)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dy.device) if nbytes else None
        p = _lib.ptr
        with _lib.device_of(dy):
            _lib.check(lib.alg_embedding_bwd(
                _lib.stream_of(dy), N, d, V, p(tokens), _INTS[tokens.dtype], p(dy), _FLOATS[dy.dtype], scale, p(grad),
                _FLOATS[dtype], p(ws), nbytes), "token_embedding backward")
        return None, *first_order("token_embedding", cotangent, grad), None, None


def token_embedding(tokens, embed, *, scale: float = 1.0, dtype: Optional[torch.dtype] = None):
    """``scale * embed[tokens]``, (*tokens.shape, d), rounded once to ``dtype`` (default: the table's).

    ``tokens`` int32 or int64 of any shape, ``embed`` (V, d) bfloat16 or float32, d a multiple of 8. A token below
    0 (padding, or ``head_sample``'s -1) has a row of zeros; one from V on has no row of the table, and
    gets NaN. Differentiable in ``embed``, once: the gradient, dense and in the table's dtype, adds up
    the tokens' rows in f32 in an order that their number alone sets, so that it is the same each time; tokens
    outside the table give nothing.
    """
    if tokens.dtype not in _INTS:
        raise ValueError(f"tokens must be int32 or int64, not {tokens.dtype}")
    if embed.dim() != 2 or embed.shape[0] == 0:
        raise ValueError("embed must be (V, d)")
    if embed.dtype not in _FLOATS:
        raise NotImplementedError(f"dtype {embed.dtype}: the gfx950 embedding takes bfloat16 or float32 tables")
    dtype = embed.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise NotImplementedError(f"dtype {dtype}: the gfx950 embedding gives bfloat16 or float32 rows")
    if tokens.device != embed.device:
        raise ValueError(f"tokens must be on {embed.device}")
    d = embed.shape[1]
    if d == 0 or d % 8:
        raise NotImplementedError(f"rows of {d}: the gfx950 embedding takes multiples of 8")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not embed.is_cuda:
        raise RuntimeError("token_embedding needs GPU tensors (no CPU fallback)")
    return _EmbeddingFn.apply(tokens, embed, float(scale), dtype)

"""From hidden states to the next tokens on MI355X: the tied head's logits, and drawing from its likelihood.

The reference's scorer takes the argmax of dense logits (src/algebraic/benchmarking.py:178-188); a serving step
draws from the algebraic likelihood p proportional to rho(z / c)^n (src/algebraic/algebraic.py:223-265) instead:

    z = head_logits(h, embed)                                  # (N, V) float32, of the step's last tokens
    tokens, logprob = head_sample(z, uniforms, n=8, c=2.0, temperature=0.8, top_p=0.95)
    x = token_embedding(tokens, embed, scale=scale)            # and on

Hand-written HIP (csrc/head_logits.hip, head_sample.hip), no CPU fallback and no gradient (training never
forms logits: ``fused_head``). Neither call reads device data on the host, so that a captured step serves any.
"""

import math

import torch

from .. import _lib
from .paged import _no_gradient

_BF16, _F32, _F64 = torch.bfloat16, torch.float32, torch.float64
_DTYPES = {_BF16: _lib.DTYPE_BF16, _F32: _lib.DTYPE_F32, _F64: _lib.DTYPE_F64}


def head_logits(h, embed):
    """The logits ``h @ embed.T``, (N, V) float32 with float32 sums.

    ``h`` (N, d) bfloat16 or float32, ``embed`` (V, d), cast to ``h``'s dtype as ``fused_head`` does (keep a copy
    of that dtype for serving: the cast reads and writes the whole table), d a multiple of 8. The order of the sums
    goes by the shapes, N among them: a row's logits may differ in their last bits between batches of different
    sizes (never between calls of one shape). No gradient.
    """
    if h.dim() != 2 or embed.dim() != 2 or h.shape[1] != embed.shape[1] or embed.shape[0] == 0:
        raise ValueError(f"h {tuple(h.shape)} and embed {tuple(embed.shape)}: (N, d) and (V, d)")
    if h.dtype is not _BF16 and h.dtype is not _F32:
        raise NotImplementedError(f"hidden dtype {h.dtype}: the gfx950 head takes bfloat16 or float32 hidden states")
    if h.device != embed.device:
        raise ValueError(f"embed must be on {h.device}")
    (N, d), V = h.shape, embed.shape[0]
    if d == 0 or d % 8:
        raise NotImplementedError(f"d = {d}: the gfx950 head takes multiples of 8")
    _no_gradient("head_logits", h, embed)
    if not h.is_cuda:
        raise RuntimeError("head_logits needs GPU tensors (no CPU fallback)")
    z = torch.empty(N, V, dtype=_F32, device=h.device)
    h, embed = _lib.aligned16(h), _lib.aligned16(embed if embed.dtype is h.dtype else embed.detach().to(h.dtype))
    p = _lib.ptr
    with _lib.device_of(h):
        _lib.check(_lib.load().alg_head_logits(_lib.stream_of(h), _DTYPES[h.dtype], N, d, V, p(h), p(embed), p(z)),
                   "head_logits")
    return z


def _setting(name, x, N, dtype, device, least):
    """A setting as the C entry point takes it: (tensor of one a row or None, value for all)."""
    if not torch.is_tensor(x):
        if not x >= least:
            raise ValueError(f"{name} must be {least} or more (got {x})")
        if dtype is torch.int32 and x // 1 != x:  # (infinity // 1 is NaN)
            raise ValueError(f"{name} must hold whole numbers")
        return None, x
    if x.dim() > 1 or (x.dim() == 1 and x.shape[0] != N):
        raise ValueError(f"{name} must be a number or a tensor ({N},)")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}")
    if dtype is torch.int32 and x.is_floating_point():
        raise ValueError(f"{name} must hold whole numbers")
    if x.dtype is not dtype:  # a top_k past int32 is past every vocabulary too, and all below 0 are alike
        x = x.clamp(0, 2 ** 31 - 1).to(dtype) if x.dtype is torch.int64 and dtype is torch.int32 else x.detach().to(dtype)
    return x.expand(N).contiguous(), 0


def head_sample(logits, uniforms, *, n: int = 8, c: float = 2.0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token a row drawn from the algebraic likelihood of ``logits`` (N, V): (tokens (N,) int64, logprob (N,) float32).

    Weights are ``rho(min(z / c, X))^(n / temperature)``, the training head's likelihood at temperature 1
    (``fused_head``'s n, c and clamp X). Of the tokens by falling logit, equal ones by their index, are kept
    the first ``top_k`` (0, or V and more: all), of those the fewest that together have ``top_p`` of their
    weight (1: all; always one), of those the ones with at least ``min_p`` of the likeliest's weight. The
    token drawn is the first kept one, by index, at which the running sum of the kept weights passes
    ``uniforms`` times their sum; ``logprob`` is the log of the probability that it had there. ``temperature`` 0 takes
    the first of the largest logits.

    ``logits`` float32 or bfloat16, rows with a contiguous last axis any distance apart, V up to 2^20; ``uniforms`` (N,)
    float32 or float64 in [0, 1) (``torch.rand``). Each setting is a number or a tensor (N,) of one a row, in which
    what is below 0 counts as 0 (but for temperatures), and a NaN ``top_p`` as 1, a NaN ``min_p`` as 0. ``c``,
    ``temperature``, ``top_p`` and ``min_p`` are taken as float32 numbers, however given (0.6 is 0.60000002...); from
    there on weights are formed in 64 bits, good to (n / temperature) 2^-44 of themselves, and
    summed in whole numbers, so that a row's token depends on nothing but the row. A
    logit of -inf is never drawn; a row without another, with a NaN, or with a temperature that is negative or
    NaN has token -1 and logprob NaN. No gradient.
    """
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be (N, V)")
    if logits.dtype is not _F32 and logits.dtype is not _BF16:
        raise NotImplementedError(f"dtype {logits.dtype}: the gfx950 sampler takes float32 or bfloat16 logits")
    (N, V), dev = logits.shape, logits.device
    if V > 1 << 20:
        raise NotImplementedError(f"{V} logits a row: the gfx950 sampler is built for up to 2^20")
    if uniforms.shape != (N,) or (uniforms.dtype is not _F32 and uniforms.dtype is not _F64):
        raise ValueError(f"uniforms must be ({N},), float32 or float64")
    if uniforms.device != dev:
        raise ValueError(f"uniforms must be on {dev}")
    if n < 1 or n & (n - 1):
        raise ValueError("n must be a power of two")
    if not math.isfinite(c) or c <= 0:
        raise ValueError("scale c must be positive and finite")
    temperature, temperature_all = _setting("temperature", temperature, N, _F32, dev, 0)
    top_k, top_k_all = _setting("top_k", top_k, N, torch.int32, dev, 0)
    top_p, top_p_all = _setting("top_p", top_p, N, _F32, dev, 0)
    min_p, min_p_all = _setting("min_p", min_p, N, _F32, dev, 0)
    _no_gradient("head_sample", logits)
    if not logits.is_cuda:
        raise RuntimeError("head_sample needs GPU tensors (no CPU fallback)")
    token = torch.empty(N, dtype=torch.int64, device=dev)
    logprob = torch.empty(N, dtype=_F32, device=dev)
    if V > 1 and logits.stride(1) != 1 or N > 1 and logits.stride(0) < V:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    lib, p = _lib.load(), _lib.ptr
    nbytes = lib.alg_head_sample_workspace_size(N, V)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _lib.device_of(logits):
        _lib.check(lib.alg_head_sample(
            _lib.stream_of(logits), N, V, p(logits), _DTYPES[logits.dtype], max(logits.stride(0), V), p(uniforms),
            _DTYPES[uniforms.dtype], int(n), float(c), p(temperature), float(temperature_all), p(top_k),
            min(int(top_k_all), 2 ** 31 - 1), p(top_p), float(top_p_all), p(min_p), float(min_p_all), p(token), p(logprob),
            p(ws), nbytes), "head_sample")
    return token, logprob

"""RMS normalisation with a learned gain on MI355X: the model's final norm ahead of the head.

``rms_norm(x, gain, eps)`` mirrors ``algebraic.rms_norm`` (src/algebraic/algebraic.py:76-83)
as the model uses it before the head (src/algebraic/model.py:208): bfloat16 rows, f32
statistics, one rounding to bfloat16; differentiable in x and the gain, with the VJP JAX's
autodiff forms for that expression. Both passes are HIP kernels (one wave per row); compose
with the head as ``fused_head(rms_norm(x, g), E, t, ...)``. No CPU fallback.

``add_rms_norm`` takes the residual stream's addition in front of a norm with it
(src/algebraic/model.py:182-187: ``x = x + ...`` and the next block's ``rms_norm``), one pass
instead of two each way; ``add_rms_norm_fp8`` leaves the norm in 8 bits with a scale per row, for
products of 8-bit operands in inference.
"""

import math

import torch

from .. import _lib
from .autograd import first_order


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gain, eps):
        lib = _lib.load()
        d = x.shape[-1]
        x2 = _lib.aligned16(x).reshape(-1, d)
        rows = x2.shape[0]
        g = None if gain is None else gain.detach().to(device=x.device, dtype=torch.float32).contiguous()
        y = torch.empty_like(x2)
        tau = torch.empty(rows, dtype=torch.float32, device=x.device)
        _lib.check(lib.alg_rms_norm_fwd(_lib.stream_of(x2), rows, d, _lib.ptr(x2), _lib.ptr(g), float(eps),
                                        _lib.ptr(y), _lib.ptr(tau)), "rms_norm")
        ctx.save_for_backward(x2, g, tau)
        ctx.gain_meta = None if gain is None else (gain.shape, gain.dtype)
        ctx.shape = x.shape
        return y.reshape(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, g, tau = ctx.saved_tensors
        lib = _lib.load()
        rows, d = x2.shape
        dy2 = _lib.aligned16(dy.to(x2.dtype)).reshape(rows, d)
        dx = torch.empty_like(x2)
        dg = torch.empty(d, dtype=torch.float32, device=x2.device) if g is not None else None
        nbytes = lib.alg_rms_norm_workspace_size(rows, d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x2.device)
        _lib.check(lib.alg_rms_norm_bwd(_lib.stream_of(x2), rows, d, _lib.ptr(x2), _lib.ptr(g), _lib.ptr(tau),
                                        _lib.ptr(dy2), _lib.ptr(dx), _lib.ptr(dg), _lib.ptr(ws), nbytes),
                   "rms_norm backward")
        dgain = None if dg is None else dg.reshape(ctx.gain_meta[0]).to(ctx.gain_meta[1])
        return dx.reshape(ctx.shape), dgain, None


def rms_norm(x, gain=None, eps: float = 1e-5):
    """``round((x rsqrt(mean(x^2) + eps)) gain)`` over the last axis of a bfloat16 GPU tensor."""
    if x.dtype != torch.bfloat16:
        raise NotImplementedError(f"dtype {x.dtype}: the gfx950 norm takes bfloat16 rows")
    if gain is not None and gain.numel() != x.shape[-1]:
        raise ValueError(f"gain must have {x.shape[-1]} entries")
    if not x.is_cuda:
        raise RuntimeError("rms_norm needs a GPU tensor (no CPU fallback)")
    return _RmsNormFn.apply(x, gain, float(eps))


_BF16, _F32 = torch.bfloat16, torch.float32
_WEIGHTS = {_BF16: _lib.DTYPE_BF16, _F32: _lib.DTYPE_F32}


class _AddRmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gain, eps):
        lib = _lib.load()
        x, residual = _lib.aligned16(x), _lib.aligned16(residual)
        d = x.shape[-1]
        rows = x.numel() // d
        g, gain_dtype = _gain_vector(gain, x.device)
        y, s = torch.empty_like(x), torch.empty_like(x)
        tau = torch.empty(rows, dtype=_F32, device=x.device)
        p = _lib.ptr
        if rows:
            with _lib.device_of(x):
                _lib.check(lib.alg_add_rms_norm_fwd(_lib.stream_of(x), rows, d, p(x), p(residual), p(g), gain_dtype, eps,
                                                    p(s), p(y), p(tau)), "add_rms_norm")
        ctx.save_for_backward(s, g, tau)
        ctx.gain_meta = None if gain is None else (gain.dtype, gain.device)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    def backward(ctx, dy, ds):
        s, g, tau = ctx.saved_tensors
        if dy is None:  # the norm was not used
            return ds, ds, None, None
        lib = _lib.load()
        d, rows = s.shape[-1], tau.shape[0]
        dy = _lib.aligned16(dy if dy.dtype is _BF16 else dy.to(_BF16))
        if ds is not None:
            ds = _lib.aligned16(ds if ds.dtype is _BF16 else ds.to(_BF16))
        dx = torch.empty_like(s)
        dg, ws, nbytes, gain_dtype = None, None, 0, 1
        if g is not None:
            gain_dtype = _WEIGHTS[g.dtype]
            if ctx.needs_input_grad[2]:
                dg = torch.empty_like(g) if rows else torch.zeros_like(g)
                nbytes = lib.alg_rms_norm_workspace_size(rows, d)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=s.device)
        p = _lib.ptr
        if rows:
            with _lib.device_of(s):
                _lib.check(lib.alg_add_rms_norm_bwd(_lib.stream_of(s), rows, d, p(s), p(g), gain_dtype, p(tau), p(dy),
                                                    p(ds), p(dx), p(dg), p(ws), nbytes), "add_rms_norm backward")
        if dg is not None:
            dtype, where = ctx.gain_meta
            if dg.dtype is not dtype or where != dg.device:
                dg = dg.to(device=where, dtype=dtype)
        dx, dg = first_order("add_rms_norm", s, dx, dg)
        return dx, dx, dg, None


def _gain_vector(gain, device):
    """The gain, f32 or bf16, contiguous and aligned, and its type's code."""
    if gain is None:
        return None, 1
    g = gain
    if g.dtype not in _WEIGHTS or g.device != device:
        g = g.detach().to(device=device, dtype=_F32)
    return _lib.aligned16(g), _WEIGHTS[g.dtype]


def _check_add(x, residual, gain, eps, what):
    if x.dtype is not _BF16 or residual.dtype is not _BF16:
        raise NotImplementedError(f"dtypes {x.dtype}, {residual.dtype}: the gfx950 norm takes bfloat16 rows")
    if x.shape != residual.shape or x.dim() == 0:
        raise ValueError(f"x {tuple(x.shape)} and residual {tuple(residual.shape)} must share a shape of rows")
    if x.device != residual.device:
        raise ValueError(f"residual must be on {x.device}")
    d = x.shape[-1]
    if gain is not None and gain.numel() != d:
        raise ValueError(f"gain must have {d} entries")
    if not (eps > 0) or not math.isfinite(eps):
        raise ValueError("eps must be positive and finite")
    if d == 0 or d % 8 or d > 4096:
        raise NotImplementedError(f"rows of {d}: the gfx950 norm takes multiples of 8 up to 4096")
    if x.numel() // d > (1 << 26) - 4:
        raise NotImplementedError(f"{x.numel() // d} rows: at most 2^26 - 4 in one launch")
    if not x.is_cuda:
        raise RuntimeError(f"{what} needs GPU tensors (no CPU fallback)")


def add_rms_norm(x, residual, gain=None, eps: float = 1e-5):
    """``(rms_norm(s, gain), s)`` with ``s = x + residual`` rounded to bfloat16, in one pass.

    bfloat16 rows of up to 4096 elements over the last axis; the norm is of the stored s.
    Differentiable in x, residual (which have the one gradient) and the gain, once: differentiating
    the norm's gradients raises.
    """
    _check_add(x, residual, gain, eps, "add_rms_norm")
    return _AddRmsNormFn.apply(x, residual, gain, float(eps))


def add_rms_norm_fp8(x, residual, gain=None, eps: float = 1e-5):
    """``(y8, scale, s)``: ``add_rms_norm`` with the norm in float8_e4m3fn and a float32 scale per
    row, (..., 1): ``y8.float() * scale`` is the norm, its largest value of the row at 448. No
    gradient (inference)."""
    _check_add(x, residual, gain, eps, "add_rms_norm_fp8")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, gain)):
        raise NotImplementedError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad() or on detached tensors")
    x, residual = _lib.aligned16(x), _lib.aligned16(residual)
    g, gain_dtype = _gain_vector(gain, x.device)
    y8 = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty_like(x)
    scale = torch.empty((*x.shape[:-1], 1), dtype=_F32, device=x.device)
    rows = scale.numel()
    p = _lib.ptr
    if rows:
        with _lib.device_of(x):
            _lib.check(_lib.load().alg_add_rms_norm_fp8(_lib.stream_of(x), rows, x.shape[-1], p(x), p(residual), p(g),
                                                        gain_dtype, float(eps), p(s), p(y8), p(scale)),
                       "add_rms_norm_fp8")
    return y8, scale, s

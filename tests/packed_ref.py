"""Float64 statement of attention over packed sequences with grouped heads, and how far a bf16
kernel's results may lie from it.

The bounds count roundings: u = 2^-8 is the most by which one rounding to bf16 moves a value,
relative to it. The kernels round the weights P, the score gradients dS, the output o (from which
the backward takes di = sum_d dO o) and their results; everything else is f32, whose share is
bounded by F32 times the sum of the magnitudes that a result adds up.

Weights of scores far below zero, in a row that the plain form serves: t = s + sqrt(s^2 + b) cancels, so that
t is off by 4 x^2 2^-24 of itself and w = t^n by n times that, which passes F32 / 2 where n x^2 > 209. There w <=
a^-n (2 |x|)^-n, and the error is at most a^-n 4 n x^2 (2 |x|)^-n 2^-24: for n = 2 that is 2^-23 a^-2 = 2^-19 low
(low = (4 a)^-n, the least mean weight of a row of that form); for n = 4, x^2 > 52 it is 256 / 52 2^-24 low, under
2^-21 low; for larger n (2 |x| / 4)^-n falls faster still (n = 32, low = (2 a)^-n: |x|^-n 128 x^2 2^-24, x^2 > 6.5).
FAR times the row's mean weight covers it: nothing to o, but to a gradient of a key whose every weight is
so small it may be much of it.
"""

import math

import torch

U = 2.0 ** -8
F32 = 1e-4
FAR = 2.0 ** -19


def rho_log(x):
    return torch.asinh(x)


def head_ref(q, k, v, sink, do=None, *, n, c, D=None, positions=None):
    """One head: q (T, D) at `positions` (default: the last T of k's), k, v (K, D), all float64, sink
    a float64 scalar tensor or None. Returns ({name: value}, {name: largest error})."""
    T, K = q.shape[0], k.shape[0]
    D = D or q.shape[1]
    alpha = 1.0 / (math.sqrt(D) * c)
    if positions is None:
        positions = torch.arange(K - T, K, device=q.device)
    x = (q @ k.T) * alpha
    dead = torch.arange(K, device=q.device)[None, :] > positions[:, None]
    a = (n * rho_log(x)).masked_fill(dead, -math.inf)
    ab = torch.full((T, 1), -math.inf, dtype=q.dtype, device=q.device) if sink is None else (n * rho_log(sink / c)).expand(T, 1)
    m = torch.maximum(a.amax(-1, keepdim=True) if K else ab, ab)
    m = torch.where(m == -math.inf, 0.0, m)  # a row without keys and sink
    w, wb = torch.exp(a - m), torch.exp(ab - m)
    z = w.sum(-1, keepdim=True) + wb
    z = torch.where(z == 0, 1.0, z)
    p, pb = w / z, wb / z
    o = p @ v
    mag_o = p @ v.abs()
    far = torch.where(dead, 0.0, FAR * p.sum(-1, keepdim=True) / (~dead).sum(-1, keepdim=True).clamp(min=1))
    tol_o = U * (mag_o + o.abs()) + F32 * mag_o + far @ v.abs()
    val, tol = {"o": o}, {"o": tol_o}
    if do is None:
        return val, tol
    r = torch.rsqrt(1 + x * x)
    di = (do * o).sum(-1, keepdim=True)
    tol_di = (do.abs() * tol_o).sum(-1, keepdim=True)
    f = n * alpha * p * r                        # dS = f (dP - di)
    ds = f * (do @ v.T - di)
    mag_ds = f * (do.abs() @ v.abs().T + (do * o).abs().sum(-1, keepdim=True))
    tol_ds = U * ds.abs() + f * tol_di + F32 * mag_ds + n * alpha * r * far * ((do @ v.T).abs() + di.abs())
    for name, value, off in (("dq", ds @ k, tol_ds @ k.abs()), ("dk", ds.T @ q, tol_ds.T @ q.abs()),
                             ("dv", p.T @ do, (U + F32) * (p.T @ do.abs()) + far.T @ do.abs())):
        val[name], tol[name] = value, off + U * value.abs()
    if sink is not None:
        rb = n / torch.sqrt(1 + (sink / c) ** 2) / c
        val["dsink"] = -(pb * di).sum() * rb
        tol["dsink"] = (pb * (tol_di + F32 * (do * o).abs().sum(-1, keepdim=True))).sum() * rb
    return val, tol


def packed_ref(q, k, v, cu, sink, do=None, *, n, c):
    """All heads and sequences: q (N, H, D), k, v (N, Hkv, D), cu a list, sink (1 or H) or None.
    Tolerances of shared heads' gradients add up over their group (one rounding counted per head)."""
    H, Hkv = q.shape[1], k.shape[1]
    G = H // Hkv
    d64 = lambda t: None if t is None else t.detach().double()  # noqa: E731
    q, k, v, do, sink = d64(q), d64(k), d64(v), d64(do), d64(sink)
    names = ["o"] if do is None else ["o", "dq", "dk", "dv"]
    shape = {"o": q, "dq": q, "dk": k, "dv": v}
    val = {m: torch.zeros_like(shape[m]) for m in names}
    tol = {m: torch.zeros_like(shape[m]) for m in names}
    if sink is not None and do is not None:
        val["dsink"], tol["dsink"] = torch.zeros(H, dtype=q.dtype, device=q.device), torch.zeros(H, dtype=q.dtype, device=q.device)
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        for h in range(H):
            j = h // G
            s = None if sink is None else sink.reshape(-1)[0 if sink.numel() == 1 else h]
            hv, ht = head_ref(q[a:b, h], k[a:b, j], v[a:b, j], s, None if do is None else do[a:b, h], n=n, c=c)
            for m in hv:
                if m == "dsink":
                    val[m][h] += hv[m]
                    tol[m][h] += ht[m]
                else:
                    at = j if m in ("dk", "dv") else h
                    val[m][a:b, at] += hv[m]
                    tol[m][a:b, at] += ht[m]
    if "dsink" in val and sink.numel() == 1:
        val["dsink"], tol["dsink"] = val["dsink"].sum().reshape(1), tol["dsink"].sum().reshape(1)
    return val, tol


def check(got, val, tol, what=""):
    """Every element within its bound (an absolute 1e-30 keeps exact zeros comparable)."""
    for name, g in got.items():
        g = g.detach().double().reshape(val[name].shape)
        assert torch.isfinite(g).all(), f"{what} {name}: not finite"
        off = (g - val[name]).abs() / (tol[name] + 1e-30)
        worst = float(off.max()) if off.numel() else 0.0
        print(f"  {what} {name}: worst {worst:.3f} of the bound", flush=True)
        assert worst <= 1.0, f"{what} {name}: {worst:.3f} times its bound"

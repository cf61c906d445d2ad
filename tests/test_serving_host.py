"""CPU: what the packed, paged and residual-norm entry points refuse, in Python and in the C ABI,
before anything is launched; and the float64 statement that the GPU tests hold them to, against
differences and against the oracle."""

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _cu(*v):
    return torch.tensor(v, dtype=torch.int32)


def _raises(error, text, call, *args, **kw):
    with pytest.raises(error, match=text):
        call(*args, **kw)


def test_packed_refusals():
    from algebraic_amd.kernels.packed import packed_flash_attention as op
    q, k, cu = _z(6, 4, 64), _z(6, 2, 64), _cu(0, 6)
    _raises(NotImplementedError, "bfloat16", op, q.float(), k.float(), k.float(), cu)
    _raises(NotImplementedError, "bfloat16", op, q, k, k.half(), cu)
    _raises(ValueError, "tokens, heads, D", op, q[0], k, k, cu)
    _raises(ValueError, "Hkv", op, q, k, _z(6, 4, 64), cu)
    _raises(ValueError, "Hkv", op, q, _z(5, 2, 64), _z(5, 2, 64), cu)
    _raises(ValueError, "evenly", op, q, _z(6, 3, 64), _z(6, 3, 64), cu)
    _raises(ValueError, "evenly", op, q, _z(6, 0, 64), _z(6, 0, 64), cu)
    _raises(NotImplementedError, "head_dim", op, _z(6, 4, 136), _z(6, 2, 136), _z(6, 2, 136), cu)
    _raises(ValueError, "int32", op, q, k, k, cu.long())
    _raises(ValueError, "cu_seqlens", op, q, k, k, cu[:0])
    _raises(ValueError, "cu_seqlens", op, q, k, k, cu[None])
    _raises(ValueError, "sink_logit", op, q, k, k, cu, torch.zeros(3))
    _raises(ValueError, "power of two", op, q, k, k, cu, n=12)
    _raises(ValueError, "positive and finite", op, q, k, k, cu, c=0.0)
    _raises(ValueError, "positive and finite", op, q, k, k, cu, c=math.inf)
    _raises(RuntimeError, "GPU", op, q, k, k, cu)


def test_paged_refusals():
    from algebraic_amd.kernels.paged import paged_append, paged_flash_attention as op
    q, kp, table, cu, kv = _z(3, 4, 64), _z(5, 2, 16, 64), torch.zeros(2, 3, dtype=torch.int32), _cu(0, 1, 3), _cu(4, 9)
    ok = (q, kp, kp, table, cu, kv)

    def bad(error, text, **change):
        args = dict(zip(("q", "kp", "vp", "table", "cu", "kv"), ok))
        extra = {m: change.pop(m) for m in ("n", "c", "sink") if m in change}
        args.update(change)
        sink = extra.pop("sink", None)
        _raises(error, text, op, *args.values(), sink, **extra)

    bad(NotImplementedError, "bfloat16", q=q.float())
    bad(ValueError, "tokens, heads, D", q=q[0])
    bad(ValueError, "evenly", q=_z(3, 3, 64))
    bad(ValueError, "share the shape", vp=_z(5, 2, 16, 128))
    bad(ValueError, "share the shape", kp=_z(5, 2, 16, 128), vp=_z(5, 2, 16, 128))
    bad(ValueError, "pages, Hkv, page, D", kp=kp[0], vp=kp[0])
    bad(NotImplementedError, "head_dim", q=_z(3, 4, 96), kp=_z(5, 2, 16, 96), vp=_z(5, 2, 16, 96))
    bad(NotImplementedError, "multiple of 16", kp=_z(5, 2, 24, 64), vp=_z(5, 2, 24, 64))
    bad(NotImplementedError, "multiple of 16", kp=kp[:0], vp=kp[:0])
    bad(NotImplementedError, "bfloat16", vp=kp.half())
    bad(ValueError, "contiguous", kp=_z(5, 2, 64, 16).transpose(2, 3), vp=kp)
    bad(ValueError, "contiguous", vp=_z(5, 2, 16, 68)[..., :64])
    bad(ValueError, "contiguous", vp=_z(1, 2, 16, 64).expand(5, -1, -1, -1))
    bad(ValueError, "page_table", table=table[:1])
    bad(ValueError, "page_table", table=table[:, :0])
    bad(ValueError, "int32", table=table.long())
    bad(ValueError, "cu_seqlens", cu=cu[:2])
    bad(ValueError, "kv_lens", kv=kv[None])
    bad(ValueError, "int32", kv=kv.float())
    bad(ValueError, "sink_logit", sink=torch.zeros(2))
    bad(ValueError, "power of two", n=3)
    bad(ValueError, "positive and finite", c=-1.0)
    bad(NotImplementedError, "no gradient", q=q.clone().requires_grad_(True))
    bad(RuntimeError, "GPU")

    k = _z(3, 2, 64)
    base = (q, k, k, kp, kp, table, cu, kv)
    cos = torch.zeros(48, 32)
    _raises(ValueError, "together", paged_append, *base, None, None, cos)
    _raises(ValueError, "cos must be", paged_append, *base, None, None, cos[:47], cos)
    _raises(ValueError, "sin must be", paged_append, *base, None, None, cos, cos[:, :31])
    _raises(ValueError, "q_gain", paged_append, *base, torch.ones(32))
    _raises(ValueError, "eps", paged_append, *base, eps=0.0)
    _raises(NotImplementedError, "no gradient", paged_append, *base, torch.ones(64, requires_grad=True))
    _raises(ValueError, "Hkv", paged_append, q, k[:2], k[:2], *base[3:])
    _raises(RuntimeError, "GPU", paged_append, *base)


def test_add_norm_refusals():
    from algebraic_amd.kernels.norm import add_rms_norm, add_rms_norm_fp8
    x = _z(3, 64)
    for op in (add_rms_norm, add_rms_norm_fp8):
        _raises(NotImplementedError, "bfloat16", op, x.float(), x)
        _raises(NotImplementedError, "bfloat16", op, x, x.half())
        _raises(ValueError, "share a shape", op, x, x[:2])
        _raises(ValueError, "share a shape", op, x, x[:1].expand(2, 64))
        _raises(ValueError, "gain", op, x, x, torch.ones(32))
        _raises(ValueError, "eps", op, x, x, None, 0.0)
        _raises(NotImplementedError, "multiples of 8", op, _z(3, 60), _z(3, 60))
        _raises(NotImplementedError, "multiples of 8", op, _z(3, 4104), _z(3, 4104))
        _raises(RuntimeError, "GPU", op, x, x)


def test_c_abi_refusals():
    from algebraic_amd import _lib
    h = _lib.load()
    P = ctypes.c_void_p

    def fails(rc, code, text):
        assert rc == code and text.encode() in h.alg_last_error(), (rc, h.alg_last_error())

    INV, UNS = _lib.ALG_ERR_INVALID, _lib.ALG_ERR_UNSUPPORTED

    def fwd(N=8, S=1, H=4, Hkv=2, D=64, q=P(16), q_ts=256, q_hs=64, k_ts=128, k_hs=64, cu=P(16), sink=None, sd=1, ns=0, c=8.0,
            n=16, o=P(16), stat=P(16), ws=None, bytes_=0):
        return h.alg_packed_attn_fwd(None, N, S, H, Hkv, D, q, q_ts, q_hs, P(16), k_ts, k_hs, P(16), k_ts, k_hs, cu, sink,
                                     sd, ns, c, n, o, stat, ws, bytes_)

    fails(fwd(N=-1), INV, "negative")
    fails(fwd(S=-1), INV, "negative")
    fails(fwd(H=5), INV, "multiple of Hkv")
    fails(fwd(Hkv=0), INV, "multiple of Hkv")
    fails(fwd(D=96), UNS, "head_dim")
    fails(fwd(H=258, q_ts=258 * 64), UNS, "at most 128")
    fails(fwd(N=1 << 30), UNS, "rows")
    fails(fwd(N=1 << 28), UNS, "rows")
    fails(fwd(S=1 << 30), UNS, "too many")
    fails(fwd(n=3), INV, "power of two")
    fails(fwd(n=1), INV, "power of two")
    fails(fwd(c=float("nan")), INV, "positive and finite")
    fails(fwd(c=1e-20), UNS, "2^-30")
    fails(fwd(cu=None), INV, "cu_seqlens")
    fails(fwd(sink=P(16), ns=3), INV, "sink_count")
    fails(fwd(sink=P(16), ns=1, sd=2), INV, "bf16 or f32")
    fails(fwd(q=None), INV, "null")
    fails(fwd(stat=None), INV, "null")
    fails(fwd(q=P(24)), INV, "aligned")
    fails(fwd(o=P(24)), INV, "aligned")
    fails(fwd(q_ts=252), INV, "strides")
    fails(fwd(k_ts=56), INV, "strides")
    fails(fwd(k_hs=8), INV, "strides")
    fails(fwd(q_hs=1 << 29), UNS, "32-bit")
    assert fwd(N=0, q=None, o=None, stat=None) == _lib.ALG_OK

    long = dict(N=4096, H=1, Hkv=1, q_ts=64, k_ts=64)  # one head: its keys go in ranges
    need = h.alg_packed_attn_fwd_workspace_size(4096, 1, 1, 1, 64)
    assert need >= 2 * 4096 * 66 * 4 and h.alg_packed_attn_fwd_workspace_size(8, 1, 4, 2, 64) == 0
    fails(fwd(**long), INV, "workspace too small")
    fails(fwd(**long, ws=P(16), bytes_=need - 1), INV, "workspace too small")
    fails(fwd(**long, ws=P(8), bytes_=need), INV, "aligned")

    def bwd(ws=P(16), bytes_=1 << 20, dsink=None, sink=None, dq=P(16), do_ts=256):
        return h.alg_packed_attn_bwd(None, 8, 1, 4, 2, 64, P(16), 256, 64, P(16), 128, 64, P(16), 128, 64, P(16), sink, 1, 1, 8.0,
                                     16, P(16), P(16), P(16), do_ts, 64, dq, P(16), P(16), dsink, 1, ws, bytes_)

    need = h.alg_packed_attn_bwd_workspace_size(8, 1, 4, 2, 64)
    assert need >= 8 * 4 * 4 and h.alg_packed_attn_bwd_workspace_size(8, 1, 5, 2, 64) == 0
    fails(bwd(bytes_=need - 1), INV, "workspace too small")
    fails(bwd(ws=None), INV, "workspace too small")
    fails(bwd(ws=P(8)), INV, "aligned")
    fails(bwd(dsink=P(16)), INV, "sink gradient")
    fails(bwd(dq=None), INV, "null")
    fails(bwd(do_ts=4), INV, "strides")

    def paged(N=1, page=16, pages=4, width=2, k_ps=2048, table=P(16), kv=P(16), ws=None, bytes_=0, vp=P(16)):
        return h.alg_paged_attn(None, N, 1, 4, 2, 64, P(16), 256, 64, P(16), k_ps, 1024, 64, vp, 2048, 1024, 64, pages, page,
                                table, width, P(16), kv, None, 1, 0, 8.0, 16, P(16), ws, bytes_)

    fails(paged(page=24), UNS, "multiple of 16")
    fails(paged(page=0), UNS, "multiple of 16")
    fails(paged(pages=0), INV, "positive")
    fails(paged(width=0), INV, "positive")
    fails(paged(width=1 << 28), UNS, "2^31")
    fails(paged(k_ps=2044), INV, "page and head strides")
    fails(paged(table=None), INV, "null")
    fails(paged(kv=None), INV, "null")
    fails(paged(vp=P(24)), INV, "aligned")
    need = h.alg_paged_attn_workspace_size(1, 1, 4, 2, 64, 1000, 16)
    assert need > 0 and h.alg_paged_attn_workspace_size(1, 1, 4, 2, 64, 2, 16) == 0
    fails(paged(width=1000), INV, "workspace too small")
    fails(paged(width=1000, ws=P(16), bytes_=need - 1), INV, "workspace too small")
    assert paged(N=0, table=None) == _lib.ALG_OK

    def append(eps=1e-5, cos=None, sin=None, rows=0, gain=None, gd=1, out=P(16), page=16):
        return h.alg_paged_append(None, 2, 1, 4, 2, 64, P(16), 256, 64, P(16), 128, 64, P(16), 128, 64, P(16), 2048, 1024, 64,
                                  P(16), 2048, 1024, 64, 4, page, P(16), 2, P(16), P(16), gain, None, gd, cos, sin, rows, eps, out)

    fails(append(eps=0.0), INV, "eps")
    fails(append(cos=P(16)), INV, "together")
    fails(append(cos=P(16), sin=P(16), rows=31), INV, "rotation tables")
    fails(append(gain=P(20)), INV, "aligned")
    fails(append(gain=P(16), gd=-1), INV, "bf16 or f32")
    fails(append(out=None), INV, "null")
    fails(append(page=8), UNS, "multiple of 16")

    fails(h.alg_add_rms_norm_fwd(None, 0, 64, P(16), P(16), None, 1, 1e-5, P(16), P(16), P(16)), INV, "positive")
    fails(h.alg_add_rms_norm_fwd(None, 1, 60, P(16), P(16), None, 1, 1e-5, P(16), P(16), P(16)), UNS, "% 8")
    fails(h.alg_add_rms_norm_fwd(None, 1, 8192, P(16), P(16), None, 1, 1e-5, P(16), P(16), P(16)), UNS, "at most")
    fails(h.alg_add_rms_norm_fwd(None, 1, 64, P(16), None, None, 1, 1e-5, P(16), P(16), P(16)), INV, "required")
    fails(h.alg_add_rms_norm_fwd(None, 1, 64, P(16), P(24), None, 1, 1e-5, P(16), P(16), P(16)), INV, "aligned")
    fails(h.alg_add_rms_norm_fwd(None, 1, 64, P(16), P(16), P(20), 1, 1e-5, P(16), P(16), P(16)), INV, "aligned")
    fails(h.alg_add_rms_norm_fp8(None, 1, 64, P(16), P(16), P(16), 7, 1e-5, P(16), P(16), P(16)), INV, "bf16 or f32")
    fails(h.alg_add_rms_norm_fp8(None, 1, 64, P(16), P(16), None, 1, 0.0, P(16), P(16), P(16)), INV, "eps")
    fails(h.alg_add_rms_norm_fp8(None, 1, 64, P(16), P(16), None, 1, 1e-5, P(16), P(16), None), INV, "required")
    fails(h.alg_add_rms_norm_bwd(None, 1, 64, P(16), None, 1, P(16), P(16), None, P(16), P(16), None, 0), INV, "gain gradient")
    fails(h.alg_add_rms_norm_bwd(None, 1, 64, P(16), P(16), 1, P(16), P(16), None, P(16), P(16), None, 0), INV, "workspace")
    fails(h.alg_add_rms_norm_bwd(None, 1, 64, P(16), None, 1, P(16), P(16), P(24), P(16), None, None, 0), INV, "aligned")


@pytest.mark.parametrize("sink", [None, 0.7, -3.0])
@pytest.mark.parametrize("n,c", [(16, 8.0), (2, 0.5), (64, 4.0)])
def test_reference_gradients_against_differences(sink, n, c):
    from packed_ref import head_ref
    gen = torch.Generator().manual_seed(n)
    rn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    T, K, D = 5, 9, 8
    x = {"dq": rn(T, D), "dk": rn(K, D), "dv": rn(K, D)}
    s = None if sink is None else torch.tensor(sink, dtype=torch.float64)
    do = rn(T, D)
    val, tol = head_ref(x["dq"], x["dk"], x["dv"], s, do, n=n, c=c)
    h = 1e-6

    def f(q, k, v, s):
        return float((head_ref(q, k, v, s, n=n, c=c)[0]["o"] * do).sum())

    for name in x:
        d = rn(*x[name].shape)
        up = f(*(x[m] + h * d if m == name else x[m] for m in x), s)
        down = f(*(x[m] - h * d if m == name else x[m] for m in x), s)
        slope = float((val[name] * d).sum())
        assert abs((up - down) / (2 * h) - slope) <= 1e-6 * float((val[name] * d).abs().sum()) + 1e-8, name
        assert (tol[name] >= 0).all()
    if s is not None:
        slope = (f(*x.values(), s + h) - f(*x.values(), s - h)) / (2 * h)
        assert abs(slope - float(val["dsink"])) <= 1e-6 * abs(slope) + 1e-8


def test_reference_matches_the_oracle():
    from oracle import attention as OA
    from packed_ref import packed_ref
    rng = np.random.default_rng(1)
    H, T, D = 2, 24, 16
    q, k, v, do = (rng.standard_normal((1, H, T, D)) for _ in range(4))
    sink = 0.3 * rng.standard_normal((1, H, 1, 1))
    want = OA.flash_attention_oracle(*(a.astype(np.float32) for a in (q, k, v)), sink.astype(np.float32), do.astype(np.float32),
                                     n=16, c=8.0, dtype="f32")
    rows = lambda a: torch.tensor(a[0].transpose(1, 0, 2))  # noqa: E731
    val, _ = packed_ref(rows(q), rows(k), rows(v), [0, T], torch.tensor(sink.reshape(-1)), rows(do), n=16, c=8.0)
    for name in ("o", "dq", "dk", "dv"):
        got, ref = val[name].numpy(), want[name][0].transpose(1, 0, 2)
        assert np.linalg.norm(got - ref) <= 1e-4 * np.linalg.norm(ref), name
    assert np.allclose(val["dsink"].numpy(), want["dsink"].reshape(-1), rtol=1e-3, atol=1e-5)


def test_float8_bytes_are_the_ones_torch_reads():
    """The 8-bit output is stored as float8_e4m3fn: 448 its largest value, no infinities."""
    t = torch.tensor([448.0, -448.0, 2.0 ** -9, 1.0], dtype=torch.float32).to(torch.float8_e4m3fn)
    assert t.view(torch.uint8).tolist() == [0x7e, 0xfe, 0x01, 0x38]

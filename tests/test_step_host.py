"""CPU: what the entry points between one token and the next refuse, in Python and in the C ABI, before anything
is launched."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

BF, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype) if dtype in (E4M3, E8M0) else torch.zeros(*shape, dtype=dtype)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _raises(error, text, call, *args, **kw):
    with pytest.raises(error, match=text):
        call(*args, **kw)


def _cache(pages=5, Hkv=2, page=16, D=64):
    p, s = _z(pages, Hkv, page, D, dtype=E4M3), _z(pages, Hkv, page, dtype=E8M0)
    return dict(kp=p, vp=p.clone(), ks=s, vs=s.clone(), table=torch.zeros(2, 3, dtype=torch.int32), cu=_i32(0, 1, 3), kv=_i32(4, 9))


def test_paged_fp8_refusals():
    from algebraic_amd import paged_append_fp8, paged_flash_attention_fp8, paged_read_fp8
    q, k = _z(3, 4, 64), _z(3, 2, 64)

    def bad(error, text, q=q, sink=None, n=16, c=16.0, attention_only=False, **change):
        cache = {**_cache(), **change}
        _raises(error, text, paged_flash_attention_fp8, q, *cache.values(), sink, n=n, c=c)
        if not attention_only:
            _raises(error, text, paged_append_fp8, q, k, k, *cache.values())
            _raises(error, text, paged_read_fp8, *cache.values(), tokens=3)

    c = _cache()
    only = dict(attention_only=True)
    bad(NotImplementedError, "bfloat16", q=q.float(), **only)
    bad(ValueError, "tokens, heads, D", q=q[0], **only)
    bad(ValueError, "evenly", q=_z(3, 3, 64), **only)
    bad(ValueError, "share the shape", vp=_z(5, 2, 16, 128, dtype=E4M3))
    bad(ValueError, "pages, Hkv, page, D", kp=c["kp"][0], vp=c["vp"][0], **only)
    bad(NotImplementedError, "head_dim", q=_z(3, 4, 96), kp=_z(5, 2, 16, 96, dtype=E4M3), vp=_z(5, 2, 16, 96, dtype=E4M3), **only)
    bad(NotImplementedError, "multiple of 16", kp=_z(5, 2, 24, 64, dtype=E4M3), vp=_z(5, 2, 24, 64, dtype=E4M3))
    bad(NotImplementedError, "multiple of 16", kp=c["kp"][:0], vp=c["vp"][:0])
    bad(NotImplementedError, "float8_e4m3fn", kp=_z(5, 2, 16, 64))
    bad(NotImplementedError, "float8_e4m3fn", vp=_z(5, 2, 16, 64, dtype=E4M3).view(torch.uint8))
    bad(NotImplementedError, "float8_e8m0fnu", ks=_z(5, 2, 16, dtype=torch.float32))
    bad(ValueError, "k_scales must be", ks=_z(5, 2, 32, dtype=E8M0))
    bad(ValueError, "v_scales must be", vs=_z(4, 2, 16, dtype=E8M0))
    bad(ValueError, "contiguous", kp=_z(5, 2, 64, 16, dtype=E4M3).transpose(2, 3))
    bad(ValueError, "contiguous", vp=_z(5, 2, 16, 72, dtype=E4M3)[..., :64])
    bad(ValueError, "contiguous", vp=_z(1, 2, 16, 64, dtype=E4M3).expand(5, -1, -1, -1))
    bad(ValueError, "contiguous", vs=_z(5, 16, 2, dtype=E8M0).transpose(1, 2))
    bad(ValueError, "contiguous", ks=_z(5, 2, 24, dtype=E8M0)[..., 8:])
    bad(ValueError, "page_table", table=c["table"][:1])
    bad(ValueError, "page_table", table=c["table"][:, :0])
    bad(ValueError, "int32", table=c["table"].long())
    bad(ValueError, "cu_seqlens", cu=c["cu"][:2])
    bad(ValueError, "kv_lens", kv=c["kv"][None])
    bad(ValueError, "sink_logit", sink=torch.zeros(2), **only)
    bad(ValueError, "power of two", n=3, **only)
    bad(ValueError, "positive and finite", c=-1.0, **only)
    bad(NotImplementedError, "no gradient", q=q.clone().requires_grad_(True), **only)
    bad(RuntimeError, "GPU")
    rest = tuple(c.values())
    cos = torch.zeros(48, 32)
    _raises(ValueError, "together", paged_append_fp8, q, k, k, *rest, None, None, cos)
    _raises(ValueError, "cos must be", paged_append_fp8, q, k, k, *rest, None, None, cos[:47], cos)
    _raises(ValueError, "sin must be", paged_append_fp8, q, k, k, *rest, None, None, cos, cos[:, :31])
    _raises(ValueError, "k_gain", paged_append_fp8, q, k, k, *rest, None, torch.ones(32))
    _raises(ValueError, "eps", paged_append_fp8, q, k, k, *rest, eps=0.0)
    _raises(NotImplementedError, "no gradient", paged_append_fp8, q, k, k, *rest, torch.ones(64, requires_grad=True))
    _raises(ValueError, "Hkv", paged_append_fp8, q, k[:2], k[:2], *rest)
    _raises(ValueError, "tokens", paged_read_fp8, *rest, tokens=-1)


def _fails(rc, code, text):
    from algebraic_amd import _lib
    assert rc == code and text in _lib.load().alg_last_error().decode(), (rc, _lib.load().alg_last_error())


def test_paged_fp8_c_abi_refusals():
    from algebraic_amd import _lib
    h, A = _lib.load(), 1 << 20  # an address that is never read: every call fails before a launch
    base = dict(N=3, S=2, H=4, Hkv=2, D=64, q=A, q_ts=256, q_hs=64, kp=A, k_ps=2048, k_hs=1024, k_ts=64, vp=A, v_ps=2048,
                v_hs=1024, v_ts=64, ks=A, ks_ps=32, ks_hs=16, vs=A, vs_ps=32, vs_hs=16, pages=5, page=16, table=A, width=3, cu=A, kv=A)
    tail = (None, 1, 0, ctypes.c_float(8.0), 16, A, None, 0)

    def attn(code, text, **change):
        a = {**base, **change}
        _fails(h.alg_paged_attn_fp8(None, *a.values(), *tail), code, text)

    attn(_lib.ALG_ERR_INVALID, "k_pages must be 16-byte aligned", kp=A + 8)
    attn(_lib.ALG_ERR_INVALID, "v_pages: strides", v_ts=72)
    attn(_lib.ALG_ERR_INVALID, "k_pages: strides", k_ps=48)
    attn(_lib.ALG_ERR_UNSUPPORTED, "passes 32-bit offsets", k_ts=1 << 25)
    attn(_lib.ALG_ERR_INVALID, "k_scales must be 16-byte aligned", ks=A + 4)
    attn(_lib.ALG_ERR_INVALID, "v_scales: strides", vs_hs=8)
    attn(_lib.ALG_ERR_INVALID, "null argument", vs=None)
    attn(_lib.ALG_ERR_UNSUPPORTED, "positive multiple of 16", page=24)
    attn(_lib.ALG_ERR_UNSUPPORTED, "at most 2^31", width=1 << 28)
    attn(_lib.ALG_ERR_UNSUPPORTED, "too many rows", N=1 << 30)
    attn(_lib.ALG_ERR_UNSUPPORTED, "head_dim", D=96)
    a = {m: base[m] for m in ("N", "S", "Hkv", "D", "kp", "k_ps", "k_hs", "k_ts", "vp", "v_ps", "v_hs", "v_ts", "ks", "ks_ps", "ks_hs",
                              "vs", "vs_ps", "vs_hs", "pages", "page", "table", "width", "cu", "kv")}
    _fails(h.alg_paged_read_fp8(None, *a.values(), A + 8, A), _lib.ALG_ERR_INVALID, "k_out and v_out")
    _fails(h.alg_paged_read_fp8(None, *a.values(), None, A), _lib.ALG_ERR_INVALID, "null argument")
    _fails(h.alg_paged_read_fp8(None, *{**a, "ks": A + 8}.values(), A, A), _lib.ALG_ERR_INVALID, "k_scales")
    append = (A, 256, 64, A, 128, 64, A, 128, 64)  # q, k, v
    b = {m: v for m, v in a.items() if m not in ("N", "S", "Hkv", "D")}
    _fails(h.alg_paged_append_fp8(None, 3, 2, 4, 2, 64, *append, *{**b, "vs": None}.values(), None, None, 0, None, None, 0,
                                  ctypes.c_float(1e-5), A), _lib.ALG_ERR_INVALID, "null argument")
    _fails(h.alg_paged_append_fp8(None, 3, 2, 4, 2, 64, *append, *{**b, "k_hs": 24}.values(), None, None, 0, None, None, 0,
                                  ctypes.c_float(1e-5), A), _lib.ALG_ERR_INVALID, "k_pages: strides")


def test_embedding_refusals():
    from algebraic_amd import token_embedding as op
    t, E = torch.zeros(3, dtype=torch.int64), _z(10, 64)
    _raises(ValueError, "int32 or int64", op, t.float(), E)
    _raises(ValueError, "int32 or int64", op, t.to(torch.int16), E)
    _raises(ValueError, "embed must be", op, t, E[0])
    _raises(ValueError, "embed must be", op, t, E[:0])
    _raises(NotImplementedError, "tables", op, t, E.half())
    _raises(NotImplementedError, "rows", op, t, E, dtype=torch.float16)
    _raises(NotImplementedError, "multiples of 8", op, t, E[:, :60])
    _raises(NotImplementedError, "multiples of 8", op, t, E[:, :0])
    _raises(ValueError, "finite", op, t, E, scale=float("inf"))
    _raises(RuntimeError, "GPU", op, t, E)


def test_logits_refusals():
    from algebraic_amd import head_logits as op
    h, E = _z(3, 64), _z(10, 64)
    _raises(ValueError, "embed", op, h[0], E)
    _raises(ValueError, "embed", op, h, E[:, :56])
    _raises(ValueError, "embed", op, h, E[:0])
    _raises(NotImplementedError, "hidden dtype", op, h.half(), E)
    _raises(NotImplementedError, "multiples of 8", op, h[:, :60], E[:, :60])
    _raises(NotImplementedError, "no gradient", op, h, E.clone().requires_grad_(True))
    _raises(RuntimeError, "GPU", op, h, E)


def test_sample_refusals():
    from algebraic_amd import head_sample as op
    z, u = torch.zeros(3, 50), torch.zeros(3)
    _raises(ValueError, "logits must be", op, z[0], u)
    _raises(ValueError, "logits must be", op, z[:, :0], u)
    _raises(NotImplementedError, "float32 or bfloat16", op, z.double(), u)
    _raises(NotImplementedError, "2\\^20", op, torch.zeros(1, 1).expand(3, (1 << 20) + 1), u)
    _raises(ValueError, "uniforms", op, z, u[:2])
    _raises(ValueError, "uniforms", op, z, u[:, None])
    _raises(ValueError, "uniforms", op, z, u.to(BF))
    _raises(ValueError, "power of two", op, z, u, n=12)
    _raises(ValueError, "positive and finite", op, z, u, c=0.0)
    for name, bad in (("temperature", -0.1), ("temperature", float("nan")), ("top_k", -1), ("top_p", -0.5), ("min_p", float("nan"))):
        _raises(ValueError, name, op, z, u, **{name: bad})
    for name in ("temperature", "top_k", "top_p", "min_p"):
        _raises(ValueError, name, op, z, u, **{name: torch.ones(2)})
        _raises(ValueError, name, op, z, u, **{name: torch.ones(3, 1)})
    _raises(ValueError, "whole numbers", op, z, u, top_k=torch.ones(3))
    _raises(NotImplementedError, "no gradient", op, z.clone().requires_grad_(True), u)
    _raises(RuntimeError, "GPU", op, z, u)


def test_step_c_abi_refusals():
    from algebraic_amd import _lib
    h, A, f = _lib.load(), 1 << 20, ctypes.c_float
    bad, no = _lib.ALG_ERR_INVALID, _lib.ALG_ERR_UNSUPPORTED
    bf, f32, f64, i32, i64 = _lib.DTYPE_BF16, _lib.DTYPE_F32, _lib.DTYPE_F64, _lib.DTYPE_I32, _lib.DTYPE_I64

    def embed(code, text, N=3, d=64, V=10, tokens=A, kind=i64, table=A, dtype=f32, y=A, y_dtype=bf):
        _fails(h.alg_embedding_fwd(None, N, d, V, tokens, kind, table, dtype, f(1.0), y, y_dtype), code, text)

    embed(bad, "must not be negative", N=-1)
    embed(bad, "must not be negative", V=0)
    embed(no, "multiples of 8", d=60)
    embed(no, "2^24", V=1 << 24)
    embed(no, "2^35", N=(1 << 24) - 1, d=1 << 16)
    embed(bad, "int32 or int64", kind=f32)
    embed(bad, "bf16 or f32", y_dtype=f64)
    embed(bad, "null argument", table=None)
    embed(bad, "16-byte aligned", y=A + 8)
    need = h.alg_embedding_bwd_workspace_size(3, 64, 10)
    assert need > 0 and h.alg_embedding_bwd_workspace_size(0, 64, 10) == 0
    _fails(h.alg_embedding_bwd(None, 3, 64, 10, A, i64, A, bf, f(1.0), A, f32, A, need - 1), bad, "workspace too small")
    _fails(h.alg_embedding_bwd(None, 3, 64, 10, A, i64, A, bf, f(1.0), None, f32, A, need), bad, "null argument")
    _fails(h.alg_embedding_bwd(None, 3, 64, 10, A, i64, A + 4, bf, f(1.0), A, f32, A, need), bad, "16-byte aligned")
    _fails(h.alg_head_logits(None, f64, 3, 64, 10, A, A, A), bad, "bf16 or f32")
    _fails(h.alg_head_logits(None, bf, 3, 60, 10, A, A, A), no, "multiples of 8")
    _fails(h.alg_head_logits(None, bf, 3, 64, 10, A, A, A + 4), bad, "16-byte aligned")
    _fails(h.alg_head_logits(None, bf, 3, 64, 10, None, A, A), bad, "null argument")
    _fails(h.alg_head_logits(None, bf, (1 << 20) + 1, 64, 10, A, A, A), no, "2^20")

    def sample(code, text, N=3, V=50, z=A, dtype=f32, stride=50, u=A, u_dtype=f32, n=8, c=2.0, T=1.0, token=A, ws=0):
        _fails(h.alg_head_sample(None, N, V, z, dtype, stride, u, u_dtype, n, f(c), None, f(T), None, 0, None, f(1.0), None, f(0.0),
                                 token, A, A, ws), code, text)

    sample(bad, "must not be negative", N=-1)
    sample(no, "2^20", V=(1 << 20) + 1)
    sample(no, "2^22", N=1 << 22)
    sample(bad, "power of two", n=12)
    sample(bad, "positive and finite", c=0.0)
    sample(bad, "bf16 or f32", dtype=f64)
    sample(bad, "f32 or f64", u_dtype=bf)
    sample(bad, "apart", stride=49)
    sample(bad, "temperature", T=-1.0)
    sample(bad, "null argument", token=None)
    need = h.alg_head_sample_workspace_size(3, 50000)
    assert need > 0 and h.alg_head_sample_workspace_size(3, 50) == h.alg_head_sample_workspace_size(0, 50000) == 0
    sample(bad, "workspace too small", V=50000, stride=50000, ws=need - 1)

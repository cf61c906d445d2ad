"""GPU: the operators between one token and the next at the edges of what they take."""

import math

import pytest

from test_step_gpu import BF, F32, F64, SETTINGS, _captured, _check_embedding, _check_sample, _gen, _logits, _sample, _within

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# --- sampling --------------------------------------------------------------------------------

@pytest.mark.parametrize("V", [300, 12301])
@pytest.mark.parametrize("T", [1e-6, 1e-10, 1e-13, 1e-16, 1e-20, 1e-30, 1e-38, 1e-45])
def test_sample_temperatures_next_to_zero(V, T):
    """Logits next to zero of either sign, closer than the weights' accuracy at such a temperature: a token, with a
    weight that is at most the largest's. log2 rho is off by 2^-44.7, and what has a weight is not under 2^-62 of the
    largest: so the token's log2 rho times n / T lies within 62 + (n / T) 2^-43.7 of the largest's (of float32 T)."""
    g, rn = _gen(V)
    N, n, c = 24, 8, 2.0
    size = 10.0 ** -torch.linspace(8, 32, N, device="cuda")[:, None]
    z = rn(N, V) * size
    u = torch.rand(N, device="cuda", generator=g)
    T = float(torch.tensor(T, dtype=F32))
    far = (torch.asinh(z.double() / c) / math.log(2)).cpu()
    for setting in (dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.3), dict(top_k=5000, top_p=0.99)):
        token, logp = _sample()(z, u, n=n, c=c, temperature=T, **setting)
        print(f"  {setting}: {token[:6].tolist()}", flush=True)
        assert (token >= 0).all() and (token < V).all() and (logp <= 0).all() and torch.isfinite(logp).all()
        token = token.cpu()
        off = (far.max(1).values - far.gather(1, token[:, None])[:, 0]) * (n / T)
        assert (off <= 62 + n / T * 2.0 ** -43.7).all(), setting
        # The largest logit alone: exact at every temperature.
        one = _sample()(z, u, n=n, c=c, temperature=T, top_k=1)
        assert torch.equal(one[0], z.argmax(1)) and not one[1].any()


@pytest.mark.parametrize("T", [0.6, 0.7, 1.3])
def test_sample_settings_are_float32_numbers(T):
    """A uniform number between the borders of a temperature and of its float32: the draw is the float32's, whether
    the temperature comes as a number or as a tensor of either type."""
    z = torch.tensor([[3.0, 2.0]], device="cuda")
    T32 = float(torch.tensor(T, dtype=F32))
    a = 8 * (math.asinh(1.5) - math.asinh(1.0))
    at, at32 = (1 / (1 + math.exp(-a / t)) for t in (T, T32))
    assert abs(at - at32) > 1e-10
    u = torch.tensor([(at + at32) / 2], dtype=F64, device="cuda")
    want = int(float(u) >= at32)
    assert want != int(float(u) >= at)
    for given in (T, torch.tensor(T, device="cuda", dtype=F32), torch.tensor([T], device="cuda", dtype=F64)):
        assert int(_sample()(z, u, temperature=given)[0]) == want
    # A c that is no float32 number likewise.
    c32 = float(torch.tensor(T, dtype=F32))
    at, at32 = (1 / (1 + math.exp(-8 * (math.asinh(3 / c) - math.asinh(2 / c)))) for c in (T, c32))
    u = torch.tensor([(at + at32) / 2], dtype=F64, device="cuda")
    assert int(_sample()(z, u, c=T)[0]) == int(float(u) >= at32) != int(float(u) >= at)


@pytest.mark.parametrize("V", [300, 12301])
def test_sample_settings_that_are_nan(V):
    """In tensors: a top_p cuts nothing, a min_p counts as 0 (as a number both are refused)."""
    g, rn = _gen(12)
    z, u = 2 * rn(3, V), torch.rand(3, device="cuda", generator=g)
    nan = torch.full((3,), math.nan, device="cuda")
    for a, b in ((dict(top_p=nan), {}), (dict(top_p=nan, top_k=20), dict(top_k=20)), (dict(min_p=nan), {}), (dict(min_p=nan, top_p=0.5), dict(top_p=0.5))):
        for x, y in zip(_sample()(z, u, **a), _sample()(z, u, **b)):
            assert torch.equal(x, y), (a, b)


# Few rows of a large vocabulary (up to 128 of more than 8192) are spread over several workgroups each; others are one
# workgroup's. The cases of test_step_gpu.py that a small vocabulary has, with a large one:

WIDE = 12301  # four tiles, the last one nearly empty, rows that start anywhere


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("what", ["any", "few values", "one value", "masked", "lowest", "huge", "signed zeros"])
def test_sample_spread_rows_of_every_kind(what, dtype, setting):
    g, rn = _gen(13)
    N = 8
    z = 2.0 * rn(N, WIDE) + 9.0 * torch.rand(N, WIDE, device="cuda", generator=g).pow(100.0)
    out = torch.rand(N, WIDE, device="cuda", generator=g) < 0.9
    if what == "few values":
        z = z.round()
    elif what == "one value":
        z = torch.full_like(z, -1.5)
    elif what == "masked":
        z = torch.where(out, -math.inf, z)
        z[0], z[0, 9000], z[1, :12288] = -math.inf, 3.0, -math.inf  # one token; the last tile alone
    elif what == "lowest":
        z = torch.where(out, torch.finfo(dtype).min, z)
    elif what == "huge":
        z = z * 10.0 ** torch.linspace(-3, 37, N, device="cuda")[:, None]
        z[1, 5], z[2, 9], z[2, 12300] = math.inf, math.inf, 3e38
        z = z.clamp(min=torch.finfo(dtype).min)
    elif what == "signed zeros":
        z = torch.where(out, 0.0, -0.0)
    # (Masses of equal tokens are multiples of one another: more borders are met, and left out.)
    _check_sample(z.to(dtype), torch.rand(N, device="cuda", generator=g), **setting, left_out=0.05 if what == "any" and dtype is F32 else 0.5)


@pytest.mark.parametrize("n,c", [(1, 2.0), (2, 0.5), (16, 8.0), (1024, 30.0)])
def test_sample_spread_rows_of_other_exponents(n, c):
    g, rn = _gen(n)
    z = 3.0 * rn(6, WIDE)
    for setting in (dict(), dict(top_p=0.7, temperature=0.9), dict(top_k=9)):
        _check_sample(z, torch.rand(6, device="cuda", generator=g), n=n, c=c, **setting)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_sample_spread_rows_without_an_answer(dtype):
    z = torch.zeros(6, WIDE, device="cuda", dtype=dtype)
    z[0], z[1, 7], z[2, :12300], z[3, 0], z[5, 12300] = -math.inf, math.nan, -math.inf, math.inf, -math.nan
    for setting in (dict(), dict(top_k=3), dict(top_p=0.5), dict(temperature=0.0)):
        token, logp = _check_sample(z, torch.full((6,), 0.3, device="cuda"), **setting, left_out=0.5)
        assert token[:3].tolist() == [-1, -1, 12300] and int(token[5]) == -1 and torch.isnan(logp[[0, 1, 5]]).all()
        assert logp[2] == 0 and int(token[3]) == 0
    T = torch.tensor([1.0, 1.0, math.nan, -1.0, math.inf, 1e-30], device="cuda")
    z = torch.arange(WIDE, device="cuda").to(dtype).expand(6, WIDE).contiguous()
    for setting in (dict(), dict(top_k=WIDE), dict(top_p=0.99999)):
        token, logp = _sample()(z, torch.full((6,), 0.999999, device="cuda"), temperature=T, **setting)
        assert token[2:4].tolist() == [-1, -1] and torch.isnan(logp[2:4]).all() and int(token[4]) >= WIDE - 3
        assert abs(float(logp[4]) + math.log(WIDE)) < 1e-4 and z[5, token[5]] == z[5].max()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_sample_spread_rows_of_any_stride(dtype):
    g, rn = _gen(14)
    wide = (2 * rn(9, WIDE + 13)).to(dtype)
    u = torch.rand(9, device="cuda", generator=g)
    for z in (wide[:, :WIDE], wide[:, 3:WIDE], wide[::2, 1:], wide.t().contiguous().t(), wide[:1, :WIDE]):
        for setting in (dict(), dict(top_p=0.9), dict(top_k=70)):
            _check_sample(z, u[:z.shape[0]], **setting, left_out=0.2 if dtype is BF else 0.05)


def _settings_of_each_row(N):
    row = torch.arange(N, device="cuda")
    return dict(temperature=torch.where(row % 5 == 0, 0.0, 0.4 + 0.005 * row), top_k=torch.where(row % 3 == 0, 0, row * 9),
                top_p=torch.where(row % 4 == 0, 1.0, 0.3 + 0.003 * row), min_p=torch.where(row % 7 == 0, 0.1, 0.0))


def test_sample_spread_rows_with_settings_of_their_own():
    g, rn = _gen(15)
    _check_sample(2.5 * rn(64, WIDE), torch.rand(64, device="cuda", generator=g), **_settings_of_each_row(64))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("V", [8193, WIDE, 50257])
def test_sample_the_same_from_one_workgroup_and_from_many(V, dtype):
    """200 rows are a workgroup each, fewer are spread: the same tokens, and the same bits of their probabilities."""
    g, rn = _gen(V)
    N = 200
    z = (2 * rn(N, V)).to(dtype)
    z[5], z[6, 4000:], z[7, 8000], z[8] = -math.inf, -math.inf, math.nan, 1.0
    u = torch.rand(N, device="cuda", generator=g)
    for setting in [*SETTINGS, _settings_of_each_row(N)]:
        whole = _sample()(z, u, **setting)
        for a, b in ((0, 3), (3, 4), (4, 12), (12, 60), (60, 188), (188, 200)):
            part = _sample()(z[a:b], u[a:b], **{k: x[a:b] if torch.is_tensor(x) else x for k, x in setting.items()})
            for x, y in zip(part, whole):
                assert torch.equal(x.nan_to_num(7.0), y[a:b].nan_to_num(7.0)), (setting, a)


def test_sample_a_share_of_equal_logits_in_the_largest_vocabulary():
    z, u = torch.zeros(2, 1 << 20, device="cuda"), torch.tensor([0.25, 0.9], device="cuda")
    _check_sample(z, u, top_k=700001, left_out=0)
    _check_sample(z.to(BF), u, top_k=3, left_out=0)


def test_sample_more_rows_than_65536():
    g, rn = _gen(16)
    z, u = 2 * rn(70001, 40), torch.rand(70001, device="cuda", generator=g)
    token, logp = _sample()(z, u, top_k=7, top_p=0.9)
    for rows in (slice(0, 9), slice(65530, 65540), slice(69992, 70001)):
        _check_sample(z[rows], u[rows], top_k=7, top_p=0.9, left_out=0.2)
        one = _sample()(z[rows], u[rows], top_k=7, top_p=0.9)
        assert torch.equal(one[0], token[rows]) and torch.equal(one[1], logp[rows])


# --- logits and embedding at the largest sizes that they take ----------------------------------

@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("N,d,V", [(1 << 20, 8, 9), (1, 8, 1 << 24), (33, 8, (1 << 24) - 5), (2, 1 << 20, 20), (70, 1 << 20, 130)])
def test_logits_at_their_largest(N, d, V, dtype):
    print(f"[logits] N{N} d{d} V{V} {dtype}", flush=True)
    g, rn = _gen(N)
    h, E = rn(N, d).to(dtype), rn(V, d).to(dtype)
    rows = torch.cat([torch.arange(min(N, 40)), torch.arange(max(0, N - 40), N)]).unique().cuda()
    cols = torch.cat([torch.arange(min(V, 500)), torch.arange(max(0, V - 500), V), torch.randint(0, V, (500,))]).unique().cuda()
    z = _logits()(h, E)[rows][:, cols]
    a, b = h[rows].double(), E[cols].double()
    _within(z, a @ b.T, (d + 1) * 2.0 ** -24 * (a.abs() @ b.abs().T), "logits")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_logits_of_many_tokens_over_a_table_past_32_bit_offsets(dtype):
    """Tokens that take the tiled products (bf16), over a table of more than 2^32 bytes."""
    V, d, N = 1200000, 2048 if dtype is BF else 1024, 600
    E = torch.zeros(V, d, dtype=dtype, device="cuda")
    E[-1], E[0], E[700000], E[1048575], E[1048576] = 1.0, 2.0, 3.0, 4.0, 5.0
    h = torch.ones(N, d, dtype=dtype, device="cuda")
    h[7] = 2.0
    z = _logits()(h, E)
    for v, x in ((-1, 1), (0, 2), (700000, 3), (1048575, 4), (1048576, 5)):
        assert (z[:7, v] == x * d).all() and (z[7, v] == 2 * x * d).all() and (z[8:, v] == x * d).all(), v
    assert int(torch.count_nonzero(z)) == 5 * N


@pytest.mark.parametrize("N,V,d", [((1 << 24) - 1, 300, 8), ((1 << 24) - 1, (1 << 24) - 1, 8), (100, 70, 1 << 16), (3000, 9, 1 << 16)])
def test_embedding_at_its_largest(N, V, d):
    print(f"[embedding] N{N} V{V} d{d}", flush=True)
    g, rn = _gen(N ^ V)
    tokens = torch.randint(-1, V + 1, (N,), device="cuda", generator=g)
    _check_embedding(tokens, rn(V, d), rn(N, d).to(BF), 0.5, BF)


# --- the 8-bit cache --------------------------------------------------------------------------

@pytest.mark.parametrize("D,heads", [(64, 16), (128, 8)])
def test_append_stores_the_bytes_of_the_64_bit_statement(D, heads):
    """Keys' bytes and scales against norm and rotation in float64, rounded to float32 and then to 8 bits, each of them
    equal: float64's own error, 2^-40 here, is allowed for by a statement a little above and below, which differ
    next to a border alone. (float32 arithmetic, off by 2^-23, would carry one key in 2^19 over one.)"""
    from algebraic_amd import paged_append_fp8
    from test_paged_fp8_gpu import E4M3, E8M0, _quantised
    from test_paged_gpu import _i32, _tables
    N, page, eps = 8000, 64, 2.0 ** -17  # (eps is a float32)
    g, rn = _gen(D)
    q, k, v = ((1.5 * rn(N, heads, D)).to(BF) for _ in range(3))
    pages = N // page
    kp, vp = (torch.zeros(pages, heads, page, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, page, dtype=torch.uint8, device="cuda") for _ in range(2))
    gq, gk = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D)
    cos, sin = _tables(N, D // 2)
    paged_append_fp8(q, k, v, kp.view(E4M3), vp.view(E4M3), ks.view(E8M0), vs.view(E8M0),
                     torch.arange(pages, dtype=torch.int32, device="cuda")[None], _i32([0, N]), _i32([N]), gq, gk, cos, sin, eps=eps)
    x = k.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gk.double()
    a, b = y.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([a * c - b * s, a * s + b * c], -1)
    off = 2.0 ** -40 * torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)
    got, scale = kp.transpose(1, 2).reshape(N, heads, D), ks.transpose(1, 2).reshape(N, heads)
    sides = [_quantised((y + t * off).float()) for t in (-1, 0, 1)]
    near = (sides[0][0] != sides[2][0]) | (sides[0][1] != sides[2][1])[..., None]
    print(f"  {int(near.sum())} of {near.numel()} next to a border", flush=True)
    assert near.sum() <= 8
    assert torch.equal(torch.where(near, sides[1][0], got), sides[1][0])
    assert torch.equal(torch.where(near.any(-1), sides[1][1], scale), sides[1][1])
    kind, unit = _quantised(v)[:2]
    assert torch.equal(vp.transpose(1, 2).reshape(N, heads, D), kind) and torch.equal(vs.transpose(1, 2).reshape(N, heads), unit)


def _held8(S, width, page, new, H, Hkv, D, seed):
    """Queries, an 8-bit cache whose every place is filled, its table, and each sequence's stored keys and values."""
    from test_paged_fp8_gpu import E4M3, E8M0, _quantised
    from test_serving_edges_gpu import _held
    q, kp, vp, table, s, _, _ = _held(S, width, page, new, H, Hkv, D, seed)
    (k8, ksc, k), (v8, vsc, v) = _quantised(kp), _quantised(vp)
    rows = lambda t, i: t[table[i].long()].transpose(1, 2).flatten(0, 1)  # noqa: E731
    return q, (k8.view(E4M3), v8.view(E4M3), ksc.view(E8M0), vsc.view(E8M0)), table, s, [rows(k, i) for i in range(S)], [rows(v, i) for i in range(S)]


def _check_attention8(q, cache, table, new, kv, sink, ks, vs, what=""):
    """Each sequence's tokens against float64; before position 0 zeros, from the table's end on NaN."""
    from algebraic_amd import paged_flash_attention_fp8
    from packed_ref import check
    from test_paged_gpu import _i32, _starts
    from test_serving_edges_gpu import _row
    at, reach = _starts(new), table.shape[1] * cache[0].shape[2]
    o = paged_flash_attention_fp8(q, *cache, table, _i32(at), _i32(kv), sink, n=16, c=8.0)
    for i, m in enumerate(new):
        pos = torch.arange(kv[i] - m, kv[i], device="cuda") if kv[i] < 1 << 30 else torch.full((m,), reach, device="cuda")
        rows = o[at[i]:at[i + 1]]
        assert not rows[pos < 0].any() and torch.isnan(rows[pos >= reach]).all(), (what, i)
        live = (pos >= 0) & (pos < reach)
        if live.any():
            held = min(kv[i], reach)
            check({"o": rows[live]}, *_row(q[at[i]:at[i + 1]][live], ks[i][:held], vs[i][:held], sink, pos[live]), f"{what} {i}")
    assert not o[at[-1]:].any()
    return o


@pytest.mark.parametrize("new,width,past,H,Hkv", [([2, 1], 2, 1, 4, 2), ([1, 1], 3, 1, 4, 2), ([40, 1], 4, 39, 4, 1), ([150, 3], 10, 40, 4, 2),
                                                  ([150, 3], 11, 150, 4, 2), ([2], 562, 1, 4, 1), ([200], 375, 50, 2, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sink", [False, True])
def test_attention8_of_lengths_past_the_table(new, width, past, H, Hkv, D, sink):
    q, cache, table, s, ks, vs = _held8(len(new), width, 16, new, H, Hkv, D, seed=sum(new) + D)
    for kv in ([16 * width + past] + [16 * width - 1] * (len(new) - 1), [(1 << 31) - 1] + [min(20, 16 * width)] * (len(new) - 1)):
        _check_attention8(q, cache, table, new, kv, s if sink else None, ks, vs, f"{new} {kv}")


@pytest.mark.parametrize("new,width", [([1, 1], 4), ([1, 1], 2000), ([1], 8192), ([2, 1], 40), ([60, 40], 4), ([150], 400)],
                         ids=["whole", "ranges", "many-ranges", "two", "chunks", "chunk-in-ranges"])
@pytest.mark.parametrize("G", [1, 4])
def test_attention8_of_a_switched_off_sink_and_rows_without_keys(new, width, G):
    q, cache, table, s, ks, vs = _held8(len(new), width, 16, new, 2 * G, 2, 64, seed=width + G)
    s[0] = s[-1] = -math.inf
    _check_attention8(q, cache, table, new, [0] * len(new), s, ks, vs)
    _check_attention8(q, cache, table, new, [new[0] // 2] + [50] * (len(new) - 1), s, ks, vs)


@pytest.mark.parametrize("S,H,Hkv,D,m", [(65, 2, 1, 64, 1), (100, 2, 1, 128, 1), (66, 2, 1, 64, 40), (70, 2, 1, 128, 40)])
def test_attention8_of_many_sequences_in_ranges(S, H, Hkv, D, m):
    from algebraic_amd import _lib
    new = [m + (i % 11 if m > 1 else 0) for i in range(S)]
    kv = [1000 + (811 * i) % 2000 for i in range(S)]
    kv[3], kv[5] = new[3], new[5]  # ranges without a key
    width = -(-max(kv) // 16)
    assert _lib.load().alg_paged_attn_fp8_workspace_size(sum(new), S, H, Hkv, D, width, 16) > 0
    q, cache, table, s, ks, vs = _held8(S, width, 16, new, H, Hkv, D, seed=S)
    _check_attention8(q, cache, table, new, kv, s, ks, vs)


@pytest.mark.parametrize("H,Hkv", [(128, 1), (64, 2), (4, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention8_of_prompts_and_single_tokens_in_one_call(H, Hkv, D):
    """The average of the rows chooses the kernel; single tokens with many heads to a key head take the prompts'."""
    for new, kv in (([300, 1, 1, 1, 1], [300, 900, 17, 1, 500]), ([1, 1, 20, 1], [1400, 3, 20, 64]), ([1, 1], [200, 31])):
        width = -(-max(kv) // 16)
        q, cache, table, s, ks, vs = _held8(len(new), width, 16, new, H, Hkv, D, seed=H + D)
        _check_attention8(q, cache, table, new, kv, s, ks, vs, f"{new}")


def test_append_and_attention8_captured_over_ranges():
    """A step of single tokens over two ranges and more, captured twice over the same buffers, whose replays alone write
    the cache; every replay is checked against the eager calls over a copy."""
    from algebraic_amd import paged_append_fp8, paged_flash_attention_fp8
    from test_paged_gpu import _i32
    S, H, Hkv, D, width, page = 3, 8, 2, 64, 130, 16
    q, cache, table, sink, _, _ = _held8(S, width, page, [1] * S, H, Hkv, D, seed=3)
    g, rn = _gen(17)
    k, v = (rn(S, Hkv, D).to(BF) for _ in range(2))
    cu, kv = _i32([0, 1, 2, 3]), _i32([1200, 2000, 1])
    copy = tuple(t.clone() for t in cache)

    def step(cache):
        return paged_flash_attention_fp8(paged_append_fp8(q, k, v, *cache, table, cu, kv), *cache, table, cu, kv, sink, n=16, c=8.0)

    graphs = _captured(lambda: step(cache))
    for t, c in zip(cache, copy):  # as before the warm-up
        t.view(torch.uint8).copy_(c.view(torch.uint8))
    for i in range(6):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        kv += 1
        want = step(copy)
        torch.cuda.synchronize()
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, copy)), i

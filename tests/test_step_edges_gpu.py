"""GPU: the operators between one token and the next at the edges of what they take."""

import math

import pytest

from test_step_gpu import BF, F32, F64, SETTINGS, _check_sample, _gen, _sample

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# --- sampling --------------------------------------------------------------------------------

@pytest.mark.parametrize("V", [300, 12301])
@pytest.mark.parametrize("T", [1e-6, 1e-10, 1e-13, 1e-16, 1e-20, 1e-30, 1e-38, 1e-45])
def test_sample_temperatures_next_to_zero(V, T):
    """Logits next to zero of either sign, closer than the weights' accuracy at such a temperature: a token, with a
    weight that is at most the largest's. log2 rho is off by 2^-44.8, and what has a weight is not under 2^-62 of the
    largest: so the token's log2 rho times n / T lies within 62 + (n / T) 2^-43.8 of the largest's (of float32 T)."""
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
        assert (off <= 62 + n / T * 2.0 ** -43.8).all(), setting
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

"""GPU: from hidden states to the next tokens and back into the model: the logits, the sampler and the embedding,
each against a float64 statement, and a serving loop of them together with the 8-bit cache."""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}  # the most by which one rounding moves a value, relative to it


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g, lambda *s: torch.randn(*s, device="cuda", generator=g)


def _within(got, want, tol, what=""):
    off = (got.double() - want).abs()
    worst = float((off / (tol + 1e-300)).max()) if off.numel() else 0.0
    print(f"  {what}: worst {worst:.3f} of the bound", flush=True)
    assert torch.isfinite(got).all() and worst <= 1.0, (what, worst)


def _captured(step, times=2):
    """`step` captured `times` over, after a warm-up on another stream: [(graph, outputs)]."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    got = []
    for _ in range(times):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        got.append((graph, out))
    torch.cuda.synchronize()
    return got


# --- logits ----------------------------------------------------------------------------------
# An f32 sum of d products in any order is off by at most d 2^-24 of the sum of their magnitudes (to first order).

def _logits():
    from algebraic_amd import head_logits
    return head_logits


def _check_logits(h, E):
    z = _logits()(h, E)
    assert z.shape == (h.shape[0], E.shape[0]) and z.dtype is F32
    a, b = h.double(), E.to(h.dtype).double()
    _within(z, a @ b.T, (h.shape[1] + 1) * 2.0 ** -24 * (a.abs() @ b.abs().T), f"logits {tuple(h.shape)} {E.shape[0]} {h.dtype}")
    return z


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [1, 5, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("d,V", [(8, 1), (64, 15), (72, 129), (1000, 1000), (2048, 513), (4104, 260)])
def test_logits(N, d, V, dtype):
    g, rn = _gen(N + d)
    _check_logits(rn(N, d).to(dtype), rn(V, d).to(dtype))


@pytest.mark.parametrize("N,d,V", [(1000, 768, 3001), (700, 200, 5000), (2049, 512, 264), (512, 1032, 2500)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logits_of_many_tokens(N, d, V, dtype):
    g, rn = _gen(N)
    _check_logits(rn(N, d).to(dtype), rn(V, d).to(dtype))


def test_logits_inputs_and_other_values():
    g, rn = _gen(1)
    h, E = rn(7, 96).to(BF), rn(50, 96)
    assert torch.equal(_check_logits(h, E), _logits()(h, E.to(BF)))  # a table of another type is cast
    assert _logits()(h[:0], E).shape == (0, 50)
    wide = rn(7, 3, 96).to(BF)
    wide[:, 1] = h
    assert torch.equal(_logits()(wide[:, 1], E), _logits()(h, E))  # a slice
    off = torch.empty(7 * 96 + 1, dtype=BF, device="cuda")[1:].view(7, 96).copy_(h)
    assert torch.equal(_logits()(off, E), _logits()(h, E))  # not on 16 bytes
    # A NaN or infinity reaches its own row or column.
    for N, d, V in ((7, 96, 50), (70, 104, 50), (300, 96, 600)):
        for dtype in (BF, F32):
            h, E = rn(N, d).to(dtype), rn(V, d).to(dtype)
            clean = _logits()(h, E)
            h[3, d - 1], E[20, 0], E[V - 1, d - 1] = math.nan, math.nan, math.inf
            z = _logits()(h, E)
            bad = torch.zeros_like(z, dtype=torch.bool)
            bad[3], bad[:, 20], bad[:, V - 1] = True, True, True
            assert torch.equal(z[~bad], clean[~bad]) and not torch.isfinite(z[bad]).any()


def test_logits_past_32_bit_offsets():
    """More than 2^31 logits (bytes of them past 2^33); a table of more than 2^32 bytes."""
    g, rn = _gen(2)
    h, E = rn(2200, 8).to(BF), rn(1000000, 8).to(BF)
    z = _logits()(h, E)
    rows, cols = torch.tensor([0, 1, 1500, 2199], device="cuda"), torch.randint(0, 1000000, (1000,), device="cuda", generator=g)
    cols[:2] = torch.tensor([0, 999999])
    a, b = h[rows].double(), E[cols].double()
    _within(z[rows][:, cols], a @ b.T, 9 * 2.0 ** -24 * (a.abs() @ b.abs().T), "wide")
    del z
    E = torch.zeros(1200000, 2048, dtype=BF, device="cuda")
    E[-1], E[0], E[700000] = 1.0, 2.0, 3.0
    h = torch.ones(3, 2048, dtype=BF, device="cuda")
    z = _logits()(h, E)
    assert (z[:, -1] == 2048).all() and (z[:, 0] == 4096).all() and (z[:, 700000] == 6144).all() and z.sum() == 3 * 12288


# --- sampling --------------------------------------------------------------------------------
# The statement works on one row in float64; where a border (of top-p's mass, of the drawn sum, of min-p) lies
# within 1e-11 of what decides there, either side is right, and the row is left out: `near`.

def _sample():
    from algebraic_amd import head_sample
    return head_sample


def _draw_ref(z, u, temperature, top_k, top_p, min_p, n, c):
    """(token, log-probability, near) of one row."""
    V = z.numel()
    z = z.double().cpu()
    if torch.isnan(z).any() or not (z > -math.inf).any() or not temperature >= 0:
        return -1, math.nan, False
    X = 0.25 * (1e38 / V) ** (1.0 / n)
    x = (z / c).clamp(max=X)
    order = torch.argsort(-x, stable=True)
    order = order[x[order] > -math.inf]
    if temperature == 0:
        return int(order[0]), 0.0, False
    a = torch.where(x.abs() > 1e100, x.sign() * (x.abs() * 2).log(), torch.asinh(x)) * (n / temperature)
    w = torch.exp(a - a[order[0]])
    near = False
    if 0 < top_k < V:
        order = order[:top_k]
    if top_p < 1:
        part = w[order].cumsum(0)
        want = top_p * float(part[-1])
        keep = int((part < want).sum()) + 1
        near |= bool(((part - want).abs() < 1e-11 * part[-1]).any())
        order = order[:max(1, min(keep, len(order)))]
    if min_p > 0:
        least = min(min_p, 1.0)
        near |= bool(((w[order] - least).abs() < 1e-11).any()) and least < 1
        order = order[w[order] >= least]
    kept = order.sort().values
    part = w[kept].cumsum(0)
    u = min(max(u, 0.0), 1.0 - 2.0 ** -53) if u == u else 0.0
    at = u * float(part[-1])
    near |= bool(((part - at).abs() < 1e-11 * part[-1]).any()) and u > 0
    i = min(int((part <= at).sum()), len(kept) - 1)
    return int(kept[i]), float(torch.log(w[kept[i]] / part[-1])), near


def _row(x, i):
    return float(x[i]) if torch.is_tensor(x) else float(x)


def _check_sample(z, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, n=8, c=2.0, left_out=0.05):
    token, logp = _sample()(z, u, n=n, c=c, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert token.dtype is torch.int64 and logp.dtype is F32 and token.shape == logp.shape == u.shape
    f = lambda x: float(torch.tensor(x, dtype=F32)) if not torch.is_tensor(x) else x  # noqa: E731  settings are f32
    skipped = 0
    for i in range(z.shape[0]):
        t, p, near = _draw_ref(z[i], float(u[i]), _row(f(temperature), i), int(_row(top_k, i)), _row(f(top_p), i), _row(f(min_p), i), n, c)
        if near:
            skipped += 1
            continue
        assert int(token[i]) == t, (i, int(token[i]), t, float(u[i]))
        # f64 up to a rounding of f32; weights that whole multiples of 2^-62 V round: 2^-40 of the largest
        assert p != p and float(logp[i]) != float(logp[i]) or abs(float(logp[i]) - p) <= 2.0 ** -23 * abs(p) + 1e-9, (i, float(logp[i]), p)
    assert skipped <= left_out * z.shape[0], skipped
    return token, logp


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_k=50, temperature=1.3), dict(top_p=0.9), dict(top_p=0.1),
            dict(min_p=0.05), dict(temperature=0.0), dict(top_k=40, top_p=0.8, min_p=0.1, temperature=0.6), dict(top_p=1e-6), dict(min_p=1.0),
            dict(top_k=1500, top_p=0.999, temperature=2.5)]


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4096, 4097, 32000, 50257])
def test_sample(V, setting):
    g, rn = _gen(V)
    N = 12 if V > 5000 else 40
    z = 2.0 * rn(N, V) + 9.0 * torch.rand(N, V, device="cuda", generator=g).pow(100.0)
    _check_sample(z, torch.rand(N, device="cuda", generator=g), **setting)


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("what", ["bf16", "few values", "one value", "masked", "huge", "signed zeros"])
def test_sample_ties_and_extreme_logits(what, setting):
    """Equal logits go by their index, whichever border they lie at; masks of -inf and of the type's lowest value."""
    g, rn = _gen(3)
    N, V = 24, 3000
    z = 2.0 * rn(N, V)
    if what == "bf16":
        z = z.to(BF)
    elif what == "few values":
        z = z.round()
    elif what == "one value":
        z = torch.full_like(z, -1.5)
    elif what == "masked":
        z = torch.where(torch.rand(N, V, device="cuda", generator=g) < 0.7, -math.inf if setting.get("top_k") else torch.finfo(F32).min, z)
        z[0], z[0, 77] = -math.inf, 3.0
    elif what == "huge":
        z = z * 10.0 ** torch.randint(-3, 39, (N, 1), device="cuda", generator=g)
        z[1, 5], z[2, 9], z[2, 20] = math.inf, math.inf, 3e38
        z[3] = z[3].clamp(min=torch.finfo(F32).min)
    else:
        z = torch.where(torch.rand(N, V, device="cuda", generator=g) < 0.5, 0.0, -0.0)
    u = torch.rand(N, device="cuda", generator=g)
    # (Masses of equal tokens are multiples of one another: more borders are met, and left out.)
    _check_sample(z, u, **setting, left_out=0.5)


@pytest.mark.parametrize("n,c", [(1, 2.0), (2, 0.5), (16, 8.0), (1024, 30.0)])
def test_sample_other_exponents(n, c):
    g, rn = _gen(n)
    z = 3.0 * rn(16, 2000)
    for setting in (dict(), dict(top_p=0.7, temperature=0.9), dict(top_k=9)):
        _check_sample(z, torch.rand(16, device="cuda", generator=g), n=n, c=c, **setting)


def test_sample_settings_of_each_row():
    g, rn = _gen(5)
    N, V = 64, 5000
    z, u = 2.5 * rn(N, V), torch.rand(N, device="cuda", generator=g)
    row = torch.arange(N, device="cuda")
    temperature = torch.where(row % 5 == 0, 0.0, 0.4 + 0.02 * row)
    top_k = torch.where(row % 3 == 0, 0, row * 3)
    top_p = torch.where(row % 4 == 0, 1.0, 0.3 + 0.01 * row)
    min_p = torch.where(row % 7 == 0, 0.1, 0.0)
    each = _check_sample(z, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    again = _sample()(z, u.double(), temperature=temperature.double(), top_k=top_k.to(torch.int32), top_p=top_p, min_p=min_p.double())
    assert torch.equal(each[0], again[0]) and torch.equal(each[1], again[1])
    # A row's result depends on nothing but the row: the same alone.
    for i in (0, 13, 63):
        one = _sample()(z[i:i + 1], u[i:i + 1], temperature=temperature[i], top_k=int(top_k[i]), top_p=float(top_p[i]), min_p=float(min_p[i]))
        assert torch.equal(one[0], each[0][i:i + 1]) and torch.equal(one[1], each[1][i:i + 1])


def test_sample_settings_below_zero():
    """In tensors, which are not read on the host: as zero."""
    g, rn = _gen(41)
    z, u = 2 * rn(5, 9001), torch.rand(5, device="cuda", generator=g)
    low = torch.tensor([-0.5, -1e30, -math.inf, -1e-30, -0.0], device="cuda")
    far = torch.tensor([-(1 << 33) + 5, -1, -(1 << 63), -(1 << 31), 0], device="cuda")
    for a, b in ((dict(top_p=low), dict(top_k=1)), (dict(top_p=low, top_k=3000), dict(top_k=1)), (dict(min_p=low), {}), (dict(top_k=far), {})):
        for x, y in zip(_sample()(z, u, **a), _sample()(z, u, **b)):
            assert torch.equal(x, y), (a, b)


def test_sample_whole_range_of_uniforms():
    """Every kept token is drawn over its own stretch of [0, 1), and no other token."""
    g, rn = _gen(6)
    V, M = 300, 4000
    z = (2.0 * rn(1, V)).expand(M, V)
    u = (torch.arange(M, device="cuda", dtype=F64) + 0.5) / M
    token, logp = _check_sample(z, u, top_p=0.8)
    assert (token[1:] >= token[:-1]).all() and abs(float(torch.exp(logp[torch.unique_consecutive(token, return_inverse=True)[1].diff(prepend=torch.tensor([-1], device="cuda")) > 0].double()).sum()) - 1) < 0.01
    ends = torch.tensor([0.0, -1.0, math.nan, 1.0, 2.0, 1.0 - 2.0 ** -53, 5e-324], dtype=F64, device="cuda")
    _check_sample(z[:7], ends, top_p=0.8, left_out=0.5)
    few = torch.tensor([-math.inf, 1.0, -math.inf, 1.0, -math.inf], device="cuda").expand(7, 5)
    got = _sample()(few, ends)[0].tolist()
    assert got == [1, 1, 1, 3, 3, 3, 1]


def test_sample_rows_without_an_answer():
    z = torch.zeros(6, 40, device="cuda")
    z[0], z[1, 7], z[2, :39], z[3, 0] = -math.inf, math.nan, -math.inf, math.inf
    for setting in (dict(), dict(top_k=3), dict(top_p=0.5), dict(temperature=0.0)):
        token, logp = _check_sample(z, torch.full((6,), 0.3, device="cuda"), **setting, left_out=0.5)  # half of 40 equal ones is a border
        assert token[:3].tolist() == [-1, -1, 39] and torch.isnan(logp[:2]).all() and logp[2] == 0 and int(token[3]) == 0
    T = torch.tensor([1.0, 1.0, math.nan, -1.0, math.inf, 1e-30], device="cuda")
    z = torch.arange(40, device="cuda").float().expand(6, 40).contiguous()
    token, logp = _sample()(z, torch.full((6,), 0.99, device="cuda"), temperature=T)
    assert token[2:4].tolist() == [-1, -1] and torch.isnan(logp[2:4]).all()
    assert int(token[4]) == 39 and abs(float(logp[4]) + math.log(40)) < 1e-6 and int(token[5]) == 39 and float(logp[5]) == 0


def test_sample_strides_and_empty():
    g, rn = _gen(8)
    for dtype in (F32, BF):
        wide = (2 * rn(9, 1013)).to(dtype)
        u = torch.rand(9, device="cuda", generator=g)
        for z in (wide[:, :1000], wide[:, 3:1000], wide[::2, 1:], wide.t().contiguous().t(), wide[:1, :1000]):
            _check_sample(z, u[:z.shape[0]], top_p=0.9)
    assert _sample()(wide[:0], u[:0])[0].shape == (0,)


def test_sample_largest_vocabulary_and_far_rows():
    g, rn = _gen(9)
    z = 2 * rn(3, 1 << 20)
    for setting in (dict(), dict(top_k=100000, top_p=0.99), dict(top_p=0.5, min_p=1e-4), dict(top_k=1 << 19)):
        _check_sample(z, torch.rand(3, device="cuda", generator=g), **setting, left_out=0.4)
    _check_sample(torch.zeros(2, 1 << 20, device="cuda"), torch.tensor([0.25, 0.9], device="cuda"), top_k=700001, left_out=1)
    base = torch.zeros(2300, 1 << 20, dtype=BF, device="cuda")  # more than 2^32 bytes
    base[:, 5], base[2299, 123456] = 4.0, 100.0
    token, logp = _sample()(base, torch.full((2300,), 0.5, device="cuda"), top_k=1)
    assert int(token[2299]) == 123456 and (token[:2299] == 5).all() and not logp.any()


def test_sample_captured_and_on_other_streams():
    g, rn = _gen(10)
    z, u = 2 * rn(20, 32000), torch.rand(20, device="cuda", generator=g)
    T, k, p = 0.5 + u, torch.arange(20, device="cuda", dtype=torch.int32) * 10, 1.0 - 0.5 * u

    def step():
        return _sample()(z, u, temperature=T, top_k=k, top_p=p, min_p=0.01)

    graphs = _captured(step)
    for i in range(4):
        z.copy_(2 * rn(20, 32000)), u.copy_(torch.rand(20, device="cuda", generator=g)), k.add_(1)
        want = step()
        torch.cuda.synchronize()
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# --- embedding -------------------------------------------------------------------------------

def _embed():
    from algebraic_amd import token_embedding
    return token_embedding


def _tokens(N, V, kind, g):
    if kind == "same":
        return torch.full((N,), V // 2, device="cuda")
    if kind == "rising":
        return (torch.arange(N, device="cuda") * V) // max(N, 1)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    if kind == "common":
        t = (V * torch.rand(N, device="cuda", generator=g, dtype=F64).pow(6)).long().clamp(max=V - 1)
    if kind == "padded":
        t[N // 3:N // 2], t[N - N // 8:] = -1, V
    return t


def _check_embedding(tokens, table, dy, scale, dtype):
    """Rows and gradient against float64: y rounded once (an f32 product and, to bf16, a rounding of it); a sum of m
    rows in f32, off by m 2^-24 of the magnitudes, times the scale, rounded to the table's type."""
    V, d = table.shape
    leaf = table.clone().requires_grad_(True)
    y = _embed()(tokens, leaf, scale=scale, dtype=dtype)
    flat = tokens.reshape(-1).long()
    ok = (flat >= 0) & (flat < V)
    rows = torch.where(ok[:, None], table.double()[flat.clamp(0, V - 1)] * scale, 0.0)
    got = y.detach().reshape(-1, d)
    assert torch.isnan(got[flat >= V]).all() and not got[flat < 0].any()
    _within(got[flat < V], rows[flat < V], ((HALF[dtype] + 2.0 ** -24) * rows.abs())[flat < V], "rows")
    grad = torch.autograd.grad(y, leaf, dy)[0]
    assert grad.dtype is table.dtype and grad.shape == table.shape
    want, mag = torch.zeros(V, d, dtype=F64, device="cuda"), torch.zeros(V, d, dtype=F64, device="cuda")
    flat_dy = dy.reshape(-1, d).double()
    want.index_add_(0, flat[ok], flat_dy[ok])
    mag.index_add_(0, flat[ok], flat_dy[ok].abs())
    count = torch.bincount(flat[ok], minlength=V).double()[:, None]
    _within(grad, want * scale, HALF[table.dtype] * (want * scale).abs() + abs(scale) * (count + 1) * 2.0 ** -24 * mag, "gradient")
    assert not grad[count[:, 0] == 0].any()
    return y.detach(), grad


@pytest.mark.parametrize("kind", ["even", "common", "same", "rising", "padded"])
@pytest.mark.parametrize("N,V,d", [(1, 1, 8), (2, 300, 64), (31, 255, 520), (32, 256, 512), (33, 257, 1032), (500, 7, 4096), (2047, 65535, 64),
                                   (2048, 65536, 8), (2049, 70001, 16), (5000, 1000, 768), (40000, 3000, 72)])
def test_embedding(N, V, d, kind):
    g, rn = _gen(N + V)
    print(f"[embedding] N{N} V{V} d{d} {kind}", flush=True)
    tokens = _tokens(N, V, kind, g)
    _check_embedding(tokens, rn(V, d), rn(N, d).to(BF), 3.3, BF)


@pytest.mark.parametrize("kind", ["even", "common", "padded"])
@pytest.mark.parametrize("N,V", [(1024, 256), (1025, 777), (4096, 65535), (4097, 50257), (16384, 1 << 18), (131072, 300), (131073, 70001),
                                 (1100000, 32000)])
def test_embedding_where_sorts_meet(N, V, kind):
    g, rn = _gen(N ^ V)
    print(f"[embedding] N{N} V{V} {kind}", flush=True)
    _check_embedding(_tokens(N, V, kind, g), rn(V, 8), rn(N, 8).to(BF), 1.5, BF)


@pytest.mark.parametrize("table", [BF, F32])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_embedding_types_and_shapes(table, dtype, ints):
    g, rn = _gen(4)
    tokens = _tokens(600, 100, "common", g).to(ints)
    E, dy = rn(100, 136).to(table), rn(20, 30, 136).to(dtype)
    _check_embedding(tokens.view(20, 30), E, dy, -0.7, dtype)
    _check_embedding(tokens.view(30, 20).t(), E, dy.transpose(0, 1).contiguous().transpose(0, 1), 1.0, dtype)
    assert _embed()(tokens[0], E).shape == (136,) and _embed()(tokens, E).dtype is table
    off = torch.empty(100 * 136 + 1, dtype=table, device="cuda")[1:].view(100, 136).copy_(E)
    assert torch.equal(_embed()(tokens, off), _embed()(tokens, E))
    # The gradient of a plain sum: one number for all of dy.
    leaf = E.clone().requires_grad_(True)
    _embed()(tokens, leaf, dtype=dtype).sum().backward()
    assert torch.equal(leaf.grad[:, 0], torch.bincount(tokens.long(), minlength=100).to(table)) and torch.equal(leaf.grad, leaf.grad[:, :1].expand(100, 136))
    none = _embed()(tokens[:0], leaf, dtype=dtype)
    assert none.shape == (0, 136) and not torch.autograd.grad(none.sum(), leaf)[0].any()


def test_embedding_far_tokens_and_offsets():
    """Tokens of any whole number; a table and rows of more than 2^32 bytes."""
    g, rn = _gen(5)
    tokens = torch.tensor([0, -1, 1 << 40, -(1 << 63), (1 << 63) - 1, 99, 100, 1 << 32], device="cuda")
    _check_embedding(tokens, rn(100, 64), rn(8, 64).to(BF), 2.0, BF)
    V, d = 1100000, 1024
    E = torch.zeros(V, d, device="cuda")
    E[V - 1], E[3] = 1.5, 2.5
    y = _embed()(torch.tensor([V - 1, 3, V - 1], device="cuda", dtype=torch.int32), E.requires_grad_(True), scale=2.0)
    assert (y[0] == 3).all() and (y[1] == 5).all() and (y[2] == 3).all()
    grad = torch.autograd.grad(y, E, torch.ones_like(y))[0]
    assert (grad[V - 1] == 4).all() and (grad[3] == 2).all() and float(grad.abs().sum()) == 6 * d
    del E, grad, y
    N = 2200000
    y = _embed()(torch.arange(N, device="cuda") % 7, torch.arange(7.0, device="cuda")[:, None].expand(7, 1024).contiguous(), dtype=BF)
    assert all((y[i] == i % 7).all() for i in (0, 1, 1048576, 2097153, N - 1))


def test_embedding_gradient_repeats_and_differentiates_once():
    g, rn = _gen(6)
    tokens, E, dy = _tokens(9000, 500, "common", g), rn(500, 768).requires_grad_(True), rn(9000, 768)
    grads = [torch.autograd.grad(_embed()(tokens, E), E, dy)[0] for _ in range(3)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])
    w = dy.clone().requires_grad_(True)
    y = _embed()(tokens, E)
    grad = torch.autograd.grad(y, E, w, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative"):
        grad.sum().backward()


def test_embedding_gradient_against_differences():
    g, rn = _gen(7)
    tokens, E, w = _tokens(50, 9, "even", g), rn(9, 16), rn(50, 16)
    leaf = E.clone().requires_grad_(True)
    grad = torch.autograd.grad((_embed()(tokens, leaf, scale=1.7) * w).sum(), leaf)[0]
    for v, k in ((0, 0), (4, 7), (8, 15)):
        step = 2.0 ** -6
        up, down = E.clone(), E.clone()
        up[v, k] += step
        down[v, k] -= step
        f = [float((_embed()(tokens, t, scale=1.7).double() * w.double()).sum()) for t in (up, down)]
        assert abs((f[0] - f[1]) / (2 * step) - float(grad[v, k])) < 1e-4 * (1 + abs(float(grad[v, k])))


def test_embedding_captured():
    """A training step's lookup and gradient captured twice over the same buffers; replays follow the tokens."""
    g, rn = _gen(8)
    tokens, dy = _tokens(3000, 700, "common", g), rn(3000, 256).to(BF)
    E = rn(700, 256).requires_grad_(True)

    def step():
        y = _embed()(tokens, E, scale=2.0, dtype=BF)
        return y.detach(), torch.autograd.grad(y, E, dy)[0]

    graphs = _captured(step)
    for i in range(4):
        tokens.copy_(_tokens(3000, 700, ("even", "same", "padded", "common")[i], g))
        dy.copy_(rn(3000, 256))
        want = step()
        torch.cuda.synchronize()
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0].nan_to_num(7.0), want[0].nan_to_num(7.0)) and torch.equal(out[1], want[1]), i


# --- together --------------------------------------------------------------------------------

def test_a_loop_from_token_to_token():
    """A one-layer model serves two requests token by token over a cache of 8 bits, captured as one graph whose
    sampled tokens are its next input; each step is checked against the eager operators, and the drawn tokens
    against the float64 statement on the step's logits."""
    from algebraic_amd import add_rms_norm, head_logits, head_sample, paged_append_fp8, paged_flash_attention_fp8, rms_norm, token_embedding
    S, H, Hkv, D, V, page, steps = 3, 4, 2, 64, 1000, 16, 6
    d = H * D
    g, rn = _gen(30)
    E = (rn(V, d) * 2 / math.sqrt(d)).to(BF)
    w, wo = (rn(d, (H + 2 * Hkv) * D) / math.sqrt(d)).to(BF), (rn(d, d) / math.sqrt(d)).to(BF)
    gq, gk, sink = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D), 0.3 * rn(H)
    angle = torch.arange(4 * page, device="cuda")[:, None] * 10000.0 ** (-torch.arange(D // 2, device="cuda") / (D // 2))
    cos, sin = angle.cos(), angle.sin()
    cache = [torch.zeros(12, Hkv, page, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)] + [
        torch.zeros(12, Hkv, page, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    table = torch.randperm(12, generator=g, device="cuda").to(torch.int32).view(S, 4)
    cu = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    kv, tokens, u = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.tensor([5, 77, 900], device="cuda"), torch.zeros(S, device="cuda")

    @torch.no_grad()
    def step():
        kv.add_(1)
        x = token_embedding(tokens, E, scale=math.sqrt(d), dtype=BF)
        q, k, v = (rms_norm(x) @ w).unflatten(1, (-1, D)).split([H, Hkv, Hkv], 1)
        q = paged_append_fp8(q, k, v, *cache, table, cu, kv, gq, gk, cos, sin)
        o = paged_flash_attention_fp8(q, *cache, table, cu, kv, sink, n=16, c=8.0)
        h, _ = add_rms_norm(o.flatten(1) @ wo, 0 * x)  # (with x a token's own row would always win)
        z = head_logits(h, E)
        new, logp = head_sample(z, u, temperature=0.8, top_k=100, top_p=0.9)
        tokens.copy_(new)
        return z, logp

    state = [t.clone() for t in (kv, tokens)]
    uniforms = torch.rand(steps, S, device="cuda", generator=g)
    eager = []
    for i in range(steps):
        u.copy_(uniforms[i])
        z, logp = step()
        for s in range(S):
            t, p, near = _draw_ref(z[s], float(u[s]), float(torch.tensor(0.8)), 100, float(torch.tensor(0.9)), 0.0, 8, 2.0)
            assert near or int(tokens[s]) == t
        eager.append((z.clone(), logp.clone(), tokens.clone()))
    assert len({tuple(t.tolist()) for _, _, t in eager}) > 1
    (graph, out), = _captured(step, 1)
    kv.copy_(state[0]), tokens.copy_(state[1])
    for t in cache[:2]:
        t.view(torch.uint8).zero_()
    for i in range(steps):
        u.copy_(uniforms[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*out, tokens), eager[i])), i

"""GPU: the paged cache of 8 bits: append, read back and attention, against the float64 statement of
tests/packed_ref.py over the values that the cache holds, and against the rule by which it holds them.

A stored row is e4m3(x 2^-e) 2^e: a value is off by at most half a step of e4m3, 2^-4 of itself or, below its
normal range, 2^-10 2^e, beside what f32 arithmetic moved x by before (the bound of the bf16 append's tests)."""

import math

import pytest

from packed_ref import check
from test_paged_gpu import _cache, _gen, _i32, _starts, _tables, _turned, _want

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _ops():
    from algebraic_amd import paged_append_fp8, paged_flash_attention_fp8, paged_read_fp8
    return paged_append_fp8, paged_flash_attention_fp8, paged_read_fp8


def _power(e):
    """2^e as float64, by its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantised(x):
    """Bytes and scale bytes (uint8) of rows of x, NaN rows as the cache holds them, and their values."""
    top = x.double().abs().amax(-1)
    m, E = torch.frexp(torch.where(top > 0, top, 1.0))
    e = (E.long() - torch.where(m <= 0.875, 9, 8)).clamp(min=-126)
    e = torch.where(top > 0, e, 0)
    unit = _power(e)
    x8 = (x.double() / unit[..., None]).to(torch.float32).to(E4M3)
    bad = ~torch.isfinite(top)
    scale = torch.where(bad, 255, e + 127).to(torch.uint8)
    return x8.view(torch.uint8), scale, torch.where(bad[..., None], math.nan, x8.double() * unit[..., None])


def _cache8(kv, new, H, Hkv, D, page, *, transposed=False, spread=True, **kw):
    """_cache's inputs with the cache in 8 bits (rows of very different sizes where `spread`), NaN
    everywhere that holds no key, and the values that it holds, whole sequence by sequence."""
    q, kp, vp, table, cu, kvl, sink, ks, vs = _cache(kv, new, H, Hkv, D, page, **kw)
    pages = kp.shape[0]
    b = {}
    for name in ("k", "v"):
        shape = (pages, page, Hkv, D) if transposed else (pages, Hkv, page, D)
        bytes_ = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda")
        b[name] = (bytes_.transpose(1, 2) if transposed else bytes_, torch.full((pages, Hkv, page), 255, dtype=torch.uint8, device="cuda"))
    for name, rows in (("k", ks), ("v", vs)):
        for s, x in enumerate(rows):
            x = x.double()
            if spread and name == "v":
                x = x * torch.exp2(torch.arange(x.shape[0], device="cuda").double() % 11 - 5)[:, None, None]
            bytes_, scale, rows[s] = _quantised(x)
            for i in range(-(-x.shape[0] // page)):
                m = slice(i * page, min((i + 1) * page, x.shape[0]))
                n = m.stop - m.start
                b[name][0][table[s, i], :, :n] = bytes_[m].transpose(0, 1)
                b[name][1][table[s, i], :, :n] = scale[m].transpose(0, 1)
    (k8, ksc), (v8, vsc) = b["k"], b["v"]
    return [q, k8.view(E4M3), v8.view(E4M3), ksc.view(E8M0), vsc.view(E8M0), table, cu, kvl, sink], ks, vs


def _check(case, new, n=16, c=8.0):
    args, ks, vs = case
    o = _ops()[1](*args, n=n, c=c)
    torch.cuda.synchronize()
    check({"o": o}, *_want(args[0], ks, vs, new, args[8], n, c))
    return o


@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 64), (4, 4, 128), (8, 2, 64), (12, 4, 128), (16, 1, 128), (32, 1, 64), (20, 1, 128)])
def test_single_tokens(H, Hkv, D, page):
    kv = [1, 2, 15, 16, 17, 31, 33, 64, 127, 200, 513, 1030]
    print(f"[paged fp8] single tokens H{H}/{Hkv} D{D} page {page}", flush=True)
    _check(_cache8(kv, [1] * len(kv), H, Hkv, D, page, seed=H + page), [1] * len(kv))


@pytest.mark.parametrize("new,kv", [([3], [3]), ([5, 1, 2], [40, 7, 300]), ([0, 4, 0, 1], [9, 70, 0, 64]), ([40], [513]),
                                    ([130, 1, 64, 7], [130, 900, 1000, 7]), ([700], [1500]), ([257, 255], [257, 1000])])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 128), (4, 1, 64), (6, 2, 128), (4, 4, 64)])
def test_chunks(new, kv, H, Hkv, D):
    print(f"[paged fp8] chunks {new} over {kv} H{H}/{Hkv} D{D}", flush=True)
    _check(_cache8(kv, new, H, Hkv, D, 48, seed=sum(new)), new)


@pytest.mark.parametrize("new,kv,H,Hkv", [([1], [9000], 4, 1), ([1], [20011], 8, 2), ([1, 1], [7000, 33], 2, 1),
                                          ([200], [6000], 2, 1), ([20], [5000], 1, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sink", [False, True])
def test_keys_split_over_workgroups(new, kv, H, Hkv, D, sink):
    print(f"[paged fp8] split {new} over {kv} H{H}/{Hkv} D{D}", flush=True)
    _check(_cache8(kv, new, H, Hkv, D, 64, seed=D, sink=sink), new)
    _check(_cache8(kv, new, H, Hkv, D, 64, seed=D, sink=sink, width=2000), new)  # ranges that hold no key


@pytest.mark.parametrize("n", [2, 8, 32, 256])
@pytest.mark.parametrize("new,kv", [([1, 1], [300, 77]), ([150], [400])])
def test_exponents(n, new, kv):
    _check(_cache8(kv, new, 4, 2, 64, 16, seed=n), new, n=n, c=8.0 if n < 256 else 100.0)


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [300, 77, 5000]), ([150, 2], [400, 90]), ([200], [5000])])
@pytest.mark.parametrize("scale", [30.0, 1e3])
def test_scores_outside_the_plain_form(new, kv, scale, sink):
    _check(_cache8(kv, new, 4, 2, 128, 16, seed=4, scale=scale, sink=sink), new)


def test_positions_without_keys_and_tokens_behind_the_last_sequence():
    attend = _ops()[1]
    args, ks, vs = _cache8([20, 5], [6, 9], 4, 2, 64, 16, seed=7)
    for s in (None, args[8]):
        o = attend(*args[:7], _i32([20, 5]), s, n=16, c=8.0)
        assert not o[6:10].any() and o[10:].any(dim=(1, 2)).all()
        assert not attend(*args[:7], _i32([0, 0]), s, n=16, c=8.0).any()
        assert not attend(*args[:7], _i32([-5, -(1 << 31)]), s, n=16, c=8.0).any()
    for new, kv in (([1, 1], [50, 70]), ([90, 1], [90, 300]), ([1], [9000])):
        o = _check(_cache8(kv, new, 4, 2, 128, 16, seed=8, extra=37), new)
        assert not o[sum(new):].any()


def test_no_sequences_and_no_tokens():
    append, attend, read = _ops()
    (q, *cache, table, cu, kv, sink), ks, vs = _cache8([20], [3], 2, 1, 64, 16, seed=15)
    k = torch.randn(3, 1, 64, device="cuda").to(BF)
    was = cache[0].view(torch.uint8).clone()
    none = (table[:0], _i32([0]), kv[:0])
    assert not append(q, k, k, *cache, *none).any() and not attend(q, *cache, *none, sink).any()
    assert not read(*cache, *none, tokens=3)[1].any()
    assert append(q[:0], k[:0], k[:0], *cache, table, _i32([0, 0]), kv).shape == (0, 2, 64)
    assert attend(q[:0], *cache, table, _i32([0, 0]), kv, sink).shape == (0, 2, 64)
    assert read(*cache, table, _i32([0, 0]), kv, tokens=0)[0].shape == (0, 1, 64)
    assert torch.equal(cache[0].view(torch.uint8), was)


def test_bad_pages_are_not_followed():
    for new, kv in (([1, 1], [500, 70]), ([90, 1], [300, 300]), ([1, 1], [9000, 100])):
        args, ks, vs = _cache8(kv, new, 4, 2, 64, 16, seed=9)
        for bad in (-1, args[1].shape[0], -(1 << 31), (1 << 31) - 1):
            broken = args[5].clone()
            broken[0, 1] = bad
            o = _ops()[1](*args[:5], broken, *args[6:], n=16, c=8.0)
            assert torch.isnan(o[:new[0]]).all() and torch.isfinite(o[new[0]:]).all(), (new, bad)


def test_positions_that_the_table_does_not_reach():
    """A sequence longer than its row of the table: the tokens within are what they would be, those behind are NaN."""
    for new, kv in (([8], [36]), ([60], [90]), ([1], [33])):
        args, ks, vs = _cache8(kv, new, 4, 2, 64, 16, seed=19)
        short = args[5][:, :2].contiguous()  # 32 positions
        first = kv[0] - new[0]
        inside = max(0, 32 - first)
        whole, o = (_ops()[1](*args[:5], t, *args[6:], n=16, c=8.0) for t in (args[5], short))
        assert torch.equal(o[:inside], whole[:inside]) and torch.isnan(o[inside:]).all()
        k, v = _ops()[2](*args[1:5], short, *args[6:8], tokens=new[0])
        assert torch.isfinite(k[:inside]).all() and torch.isnan(k[inside:]).all() and torch.isnan(v[inside:]).all()


def test_storage_order_strides_and_shared_pages():
    new, kv = [1, 40, 3], [100, 90, 33]
    a, ks, vs = _cache8(kv, new, 8, 2, 64, 32, seed=10)
    b, _, _ = _cache8(kv, new, 8, 2, 64, 32, seed=10, transposed=True)
    assert b[1].stride() != a[1].stride()
    one, two = _check((a, ks, vs), new), _check((b, ks, vs), new)
    assert torch.equal(one, two)
    # Queries as a slice of a projection; heads before pages in storage, scales too.
    proj = torch.randn(a[0].shape[0], 3, 8, 64, device="cuda").to(BF)
    proj[:, 1] = a[0]
    moved = [t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(t.dtype) for t in a[1:5]]
    assert moved[2].stride(1) > moved[2].stride(0)
    assert torch.equal(_ops()[1](proj[:, 1], *moved, *a[5:], n=16, c=8.0), one)
    for x, y in zip(_ops()[2](*moved, *a[5:8], tokens=44), _ops()[2](*b[1:5], *a[5:8], tokens=44)):
        assert torch.equal(x, y)
    # Two sequences over the same pages.
    o = _ops()[1](a[0][:2], *a[1:5], a[5][[0, 0]], _i32([0, 1, 2]), _i32([100, 100]), a[8], n=16, c=8.0)
    check({"o": o}, *_want(a[0][:2], [ks[0], ks[0]], [vs[0], vs[0]], [1, 1], a[8], 16, 8.0))


def test_a_cache_past_32_bit_offsets():
    """5 GB of keys: the used pages lie beyond 2^31 bytes and beyond 2^32 bytes."""
    append, attend, read = _ops()
    page, Hkv, D = 128, 8, 128
    pages = 5 * (1 << 30) // (page * Hkv * D)
    g, rn = _gen(11)
    kp, vp = (torch.empty(pages, Hkv, page, D, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.empty(pages, Hkv, page, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2))
    ids = [pages - 1, pages // 2, 0, pages - 2]
    q, k, v = (rn(400, h, D).to(BF) for h in (16, Hkv, Hkv))
    rest = (kp, vp, ks, vs, _i32([ids]), _i32([0, 400]), _i32([400]))
    qa = append(q, k, v, *rest)
    kn, vn = read(*rest, tokens=400)
    assert torch.equal(vn.double(), _quantised(v)[2])
    sink = 0.3 * rn(16)
    check({"o": attend(qa, *rest, sink, n=16, c=8.0)}, *_want(qa, [kn], [vn], [400], sink, 16, 8.0))
    o = attend(qa[399:], *rest[:5], _i32([0, 1]), rest[6], sink, n=16, c=8.0)
    check({"o": o}, *_want(qa[399:], [kn], [vn], [1], sink, 16, 8.0))


def test_many_sequences():
    attend = _ops()[1]
    for S in (64, 65, 4097):
        kv = [1 + (7 * i) % 19 for i in range(65)]
        args, ks, vs = _cache8(kv, [1] * 65, 2, 1, 64, 16, seed=S)
        pick = [i % 65 for i in range(S)]
        o = attend(args[0][pick], *args[1:5], args[5][pick], _i32(list(range(S + 1))), args[7][pick], args[8], n=16, c=8.0)
        want, tol = _want(args[0], ks, vs, [1] * 65, args[8], 16, 8.0)
        m = min(S, 65)
        check({"o": o[:m]}, {"o": want["o"][:m]}, {"o": tol["o"][:m]})
        assert torch.equal(o, o[:m][pick]) if S > 64 else True


# --- append and read back -----------------------------------------------------------------------

def _check_stored(x, tol, bytes_, scale):
    """Stored rows against the float64 rows x, known to `tol`."""
    e = scale.long() - 127
    unit = _power(e)
    got = bytes_.view(E4M3).double() * unit[..., None]
    top, slack = x.abs().amax(-1), tol.amax(-1)
    assert (top - slack <= 448 * unit).all() and ((top + slack > 224 * unit) | (e == -126) | (top == 0)).all()
    check({"stored": got}, {"stored": x}, {"stored": 2.0 ** -4 * (x.abs() + tol) + 2.0 ** -10 * unit[..., None] + tol})
    return got


@pytest.mark.parametrize("H,Hkv,D,page", [(4, 2, 64, 16), (3, 1, 128, 48), (16, 16, 128, 64), (40, 8, 64, 32)])
@pytest.mark.parametrize("gain", [None, torch.float32, BF])
@pytest.mark.parametrize("rotate", [True, False])
def test_append(H, Hkv, D, page, gain, rotate):
    append, _, read = _ops()
    new, kv, tail = [1, 70, 0, 5, 1], [40, 70, 9, 130, 1], 3
    g, rn = _gen(D + page)
    N, m, width = sum(new) + tail, sum(new), 10
    q, k, v = ((2 * rn(N, h, D)).to(BF) for h in (H, Hkv, Hkv))
    v = v * torch.exp2(torch.randint(-40, 40, (N, Hkv, 1), device="cuda", generator=g)).to(BF)
    v[2], v[3, 0] = 0, torch.linspace(-448, 448, D, device="cuda").to(BF)  # rows of zeros, and at the border
    v[4, 0] = torch.where(torch.arange(D, device="cuda") == 1, 2.0 ** -126, 0.0).to(BF)  # below the least scale's reach
    table = torch.randperm(5 * width, generator=g, device="cuda").to(torch.int32).view(5, width)
    kp, vp = (torch.full((5 * width, Hkv, page, D), 7, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((5 * width, Hkv, page), 9, dtype=torch.uint8, device="cuda") for _ in range(2))
    cache = (kp.view(E4M3), vp.view(E4M3), ks.view(E8M0), vs.view(E8M0))
    cos, sin = _tables(width * page, D // 2) if rotate else (None, None)
    gq, gk = ((1 + 0.2 * rn(D)).to(gain) for _ in range(2)) if gain else (None, None)
    print(f"[append fp8] H{H}/{Hkv} D{D} page {page} gain {gain} rotate {rotate}", flush=True)
    args = (table, _i32(_starts(new)), _i32(kv))
    qo = append(q, k, v, *cache, *args, gq, gk, cos, sin)
    torch.cuda.synchronize()
    pos = torch.tensor([kv[s] - new[s] + t for s in range(5) for t in range(new[s])], device="cuda")
    seq = torch.tensor([s for s in range(5) for _ in range(new[s])], device="cuda")
    y, tol = _turned(q[:m], gq, cos, sin, pos)
    check({"q": qo[:m]}, {"q": y}, {"q": tol})
    assert not qo[m:].any()
    at = table.long()[seq, pos // page]
    y, tol = _turned(k[:m], gk, cos, sin, pos)
    k_is = _check_stored(y, tol - 2.0 ** -8 * y.abs(), kp[at, :, pos % page], ks[at, :, pos % page])  # no rounding to bf16
    v_is = _check_stored(v[:m].double(), torch.zeros_like(v[:m]).double(), vp[at, :, pos % page], vs[at, :, pos % page])
    assert torch.equal(vs[at, :, pos % page], _quantised(v[:m])[1]) and torch.equal(v_is, _quantised(v[:m])[2])
    # Read back: the same values, but those under 2^-126.
    kr, vr = read(*cache, *args, tokens=N)
    assert torch.equal(kr[:m].double(), k_is) and torch.equal(vr[:m].double(), torch.where(v_is.abs() < 2.0 ** -126, 0.0, v_is))
    assert not kr[m:].any() and not vr[m:].any()
    # Nothing else is written.
    kp[at, :, pos % page], vp[at, :, pos % page], ks[at, :, pos % page], vs[at, :, pos % page] = 7, 7, 9, 9
    assert (kp == 7).all() and (vp == 7).all() and (ks == 9).all() and (vs == 9).all()


def test_append_out_of_range_places():
    append, _, read = _ops()
    D, page = 64, 16
    g, rn = _gen(2)
    q, k, v = (rn(6, h, D).to(BF) for h in (2, 1, 1))
    kp, vp = (torch.full((4, 1, page, D), 7, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((4, 1, page), 9, dtype=torch.uint8, device="cuda") for _ in range(2))
    rest = (kp.view(E4M3), vp.view(E4M3), ks.view(E8M0), vs.view(E8M0), _i32([[0, 1], [2, 3], [-1, 4]]), _i32([0, 2, 4, 6]), _i32([1, 33, 17]))
    qo = append(q, k, v, *rest)
    assert not qo[0].any() and qo[1].any() and qo[2].any() and not qo[3].any() and qo[4:].any(dim=(1, 2)).all()
    kr, vr = read(*rest, tokens=6)
    assert torch.equal(vr[1:3].double(), _quantised(v[1:3])[2]) and not vr[0].any() and not kr[0].any()
    assert torch.isnan(vr[3:]).all() and torch.isnan(kr[3:]).all()
    for b, s in ((kp, ks), (vp, vs)):
        b[0, :, 0] = b[3, :, 15] = 7
        s[0, :, 0] = s[3, :, 15] = 9
        assert (b == 7).all() and (s == 9).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("chunk", [5, 90])
def test_values_that_are_not_finite_reach_the_tokens_that_see_them(D, chunk):
    """A NaN or infinity in a key or value: NaN for the tokens at and behind it at the heads that read
    it, the others as without it, also in the same call."""
    append, attend, read = _ops()
    H, Hkv, page, held = 4, 2, 16, 40 + chunk
    g, rn = _gen(31)
    q, k, v = (rn(held, h, D).to(BF) for h in (H, Hkv, Hkv))
    table, at = _i32([list(range(9))]), 40 + chunk // 2
    for name, what in (("k", math.nan), ("v", math.nan), ("v", math.inf), ("k", -math.inf)):
        out = []
        for put in (False, True):
            cache = [torch.zeros(9, Hkv, page, D, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)] + [
                torch.zeros(9, Hkv, page, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2)]
            k2, v2 = k.clone(), v.clone()
            if put:
                (k2 if name == "k" else v2)[at, 1, 3] = what
            append(q, k2, v2, *cache, table, _i32([0, held]), _i32([held]))
            out.append(attend(q[40:], *cache, table, _i32([0, chunk]), _i32([held]), None, n=16, c=8.0))
            kr, vr = read(*cache, table, _i32([0, held]), _i32([held]), tokens=held)
            if not put:
                want, tol = _want(q[40:], [kr], [vr], [chunk], None, 16, 8.0)
            else:
                bad = torch.isnan(kr if name == "k" else vr)
                assert bad[at, 1].all() and bad.sum() == D and torch.isfinite(vr if name == "k" else kr).all()
        clean, got = out
        n = at - 40
        # (A tile with a NaN row takes the careful form of the weights: other roundings, the same bound.)
        for rows, heads in ((slice(None, n), slice(None)), (slice(n, None), slice(0, 2))):
            for o in (clean, got):
                check({"o": o[rows, heads]}, {"o": want["o"][rows, heads]}, {"o": tol["o"][rows, heads]}, f"{name} {what}")
        assert torch.isnan(got[n:, 2:]).all(), (name, what)


def test_captured_steps_follow_the_lengths():
    """Append, read back and attention captured once, with two graphs of the same buffers; replayed as
    the sequences grow by a token, between eager calls on other inputs."""
    append, attend, read = _ops()
    g, rn = _gen(12)
    q, k, v = (rn(3, h, 64).to(BF) for h in (4, 2, 2))
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20)
    bytes_ = [torch.zeros(60, 2, 16, 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((60, 2, 16), 127, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for b in bytes_:
        b.copy_(torch.randint(0, 126, b.shape, device="cuda", generator=g, dtype=torch.uint8))
    cache = [b.view(E4M3) for b in bytes_] + [s.view(E8M0) for s in scales]
    cu, kv, sink = _i32([0, 1, 2, 3]), _i32([30, 200, 47]), 0.3 * rn(4)

    def step():
        o = attend(append(q, k, v, *cache, table, cu, kv), *cache, table, cu, kv, sink, n=16, c=8.0)
        return [o, *read(*cache, table, cu, kv, tokens=3)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    torch.cuda.synchronize()
    for i in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        kv += 1
        want, was = step(), [t.clone() for t in bytes_ + scales]
        for t, w in zip(bytes_ + scales, was):
            t.add_(1)
            t.copy_(w)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i % 2], want)), i
        assert all(torch.equal(a, b) for a, b in zip(bytes_ + scales, was)), i


def test_repeats_and_other_streams():
    args, ks, vs = _cache8([5000, 31], [1, 1], 8, 2, 128, 16, seed=13)
    first = _ops()[1](*args, n=16, c=8.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [_ops()[1](*args, n=16, c=8.0) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        assert torch.equal(o, first)

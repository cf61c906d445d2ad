"""GPU: attention of new tokens over a paged cache and the append that fills it, against the float64
statement of tests/packed_ref.py, and a serving run of the operators together."""

import math

import pytest

from packed_ref import F32, U, check, head_ref, packed_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _ops():
    from algebraic_amd.kernels.paged import paged_append, paged_flash_attention
    return paged_append, paged_flash_attention


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g, lambda *s: torch.randn(*s, device="cuda", generator=g)


def _norm(t):
    return t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()


def _cache(kv, new, H, Hkv, D, page, *, seed=0, scale=1.0, extra=0, sink=True, transposed=False, width=None):
    """Inputs of a call: whole per-sequence keys and values, and a cache of shuffled pages that holds
    them, NaN everywhere else; table entries behind a sequence's end are out of range."""
    g, rn = _gen(seed)
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    shape = (pages, page, Hkv, D) if transposed else (pages, Hkv, page, D)
    kp, vp = (torch.full(shape, float("nan"), dtype=BF, device="cuda") for _ in range(2))
    if transposed:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    table = torch.full((len(kv), width or max(max(need), 1)), 1 << 30, dtype=torch.int32)
    ks, vs = [], []
    for s, n in enumerate(kv):
        k, v = (_norm(rn(n, Hkv, D)) * scale).to(BF), rn(n, Hkv, D).to(BF)
        ks.append(k)
        vs.append(v)
        for i in range(need[s]):
            id = order.pop()
            table[s, i] = id
            m = min(page, n - i * page)
            kp[id, :, :m] = k[i * page:i * page + m].transpose(0, 1)
            vp[id, :, :m] = v[i * page:i * page + m].transpose(0, 1)
    q = _norm(rn(sum(new) + extra, H, D)).to(BF)
    return q, kp, vp, table.cuda(), _i32(_starts(new)), _i32(kv), 0.3 * rn(H) if sink else None, ks, vs


def _want(q, ks, vs, new, sink, n, c):
    val, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    H = q.shape[1]
    at = 0
    for k, v, m in zip(ks, vs, new):
        G = H // k.shape[1]
        for h in range(H if m else 0):
            s = None if sink is None else sink[h].double()
            pos = torch.arange(k.shape[0] - m, k.shape[0], device="cuda")
            hv, ht = head_ref(q[at:at + m, h].double(), k[:, h // G].double(), v[:, h // G].double(), s, n=n, c=c, positions=pos)
            val[at:at + m, h], tol[at:at + m, h] = hv["o"], ht["o"]
        at += m
    return {"o": val}, {"o": tol}


def _check(case, new, n=16, c=8.0):
    q, kp, vp, table, cu, kv, sink, ks, vs = case
    o = _ops()[1](q, kp, vp, table, cu, kv, sink, n=n, c=c)
    torch.cuda.synchronize()
    check({"o": o}, *_want(q, ks, vs, new, sink, n, c))
    return o


@pytest.mark.parametrize("page", [16, 48, 64, 128])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 64), (4, 4, 128), (8, 2, 64), (12, 4, 128), (16, 1, 128), (32, 1, 64), (20, 1, 128)])
def test_single_tokens(H, Hkv, D, page):
    kv = [1, 2, 15, 16, 17, 31, 33, 64, 127, 200, 513, 1030]
    print(f"[paged] single tokens H{H}/{Hkv} D{D} page {page}", flush=True)
    _check(_cache(kv, [1] * len(kv), H, Hkv, D, page, seed=H + page), [1] * len(kv))


@pytest.mark.parametrize("new,kv", [([3], [3]), ([5, 1, 2], [40, 7, 300]), ([0, 4, 0, 1], [9, 70, 0, 64]), ([40], [513]),
                                    ([130, 1, 64, 7], [130, 900, 1000, 7]), ([700], [1500]), ([257, 255], [257, 1000])])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 128), (4, 1, 64), (6, 2, 128)])
def test_chunks(new, kv, H, Hkv, D):
    print(f"[paged] chunks {new} over {kv} H{H}/{Hkv} D{D}", flush=True)
    _check(_cache(kv, new, H, Hkv, D, 48, seed=sum(new)), new)


@pytest.mark.parametrize("new,kv,H,Hkv", [([1], [9000], 4, 1), ([1], [20011], 8, 2), ([1, 1], [7000, 33], 2, 1),
                                          ([200], [6000], 2, 1), ([20], [5000], 1, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sink", [False, True])
def test_keys_split_over_workgroups(new, kv, H, Hkv, D, sink):
    print(f"[paged] split {new} over {kv} H{H}/{Hkv} D{D}", flush=True)
    _check(_cache(kv, new, H, Hkv, D, 64, seed=D, sink=sink), new)
    # The same over a table far wider than the sequences: ranges that hold no key at all.
    _check(_cache(kv, new, H, Hkv, D, 64, seed=D, sink=sink, width=2000), new)


@pytest.mark.parametrize("n", [2, 8, 32, 256])
@pytest.mark.parametrize("new,kv", [([1, 1], [300, 77]), ([150], [400])])
def test_exponents(n, new, kv):
    _check(_cache(kv, new, 4, 2, 64, 16, seed=n), new, n=n, c=8.0 if n < 256 else 100.0)


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [300, 77, 5000]), ([150, 2], [400, 90]), ([200], [5000])])
@pytest.mark.parametrize("scale", [30.0, 1e3])
def test_scores_outside_the_plain_form(new, kv, scale, sink):
    _check(_cache(kv, new, 4, 2, 128, 16, seed=4, scale=scale, sink=sink), new)


def test_large_scores_late_in_a_row():
    """A wave that has summed blocks in the plain form meets a large score and goes on from there;
    one whose scores are all far below; the same with the large score in another key range."""
    for at in (700, 3999):
        q, kp, vp, table, cu, kv, sink, ks, vs = _cache([4000, 4000], [1, 1], 2, 1, 64, 16, seed=6)
        with torch.no_grad():
            ks[0][at] = (40 * q[0, 0]).to(BF)
            kp[table[0, at // 16], 0, at % 16] = ks[0][at, 0]
            ks[1][:] = (-3 * q[1, 0].float()).to(BF)
            for i in range(250):
                kp[table[1, i], 0] = ks[1][0, 0]
        _check((q, kp, vp, table, cu, kv, sink, ks, vs), [1, 1])
        _check((q, kp, vp, table, cu, kv, None, ks, vs), [1, 1])


def test_more_new_tokens_than_keys_and_rows_without_keys():
    """Positions before 0 hold nothing: zeros, with and without a sink; a sequence that holds no key."""
    append, attend = _ops()
    q, kp, vp, table, cu, kv, sink, ks, vs = _cache([20, 5], [6, 9], 4, 2, 64, 16, seed=7)
    for s in (None, sink):
        o = attend(q, kp, vp, table, cu, _i32([20, 5]), s, n=16, c=8.0)
        assert not o[6:10].any() and o[10:].any(dim=(1, 2)).all()
        want, tol = _want(torch.cat([q[:6], q[10:]]), ks, vs, [6, 5], s, 16, 8.0)
        check({"o": torch.cat([o[:6], o[10:]])}, want, tol)
        assert not attend(q, kp, vp, table, cu, _i32([0, 0]), s, n=16, c=8.0).any()
        assert not attend(q, kp, vp, table, cu, _i32([-5, -(1 << 31)]), s, n=16, c=8.0).any()
        o = attend(q[:2], kp, vp, table, _i32([0, 1, 2]), _i32([0, 5]), s, n=16, c=8.0)  # single tokens
        assert not o[0].any() and o[1].any()


def test_tokens_behind_the_last_sequence():
    for new, kv in (([1, 1], [50, 70]), ([90, 1], [90, 300]), ([1], [9000])):
        case = _cache(kv, new, 4, 2, 128, 16, seed=8, extra=37)
        o = _check(case, new)
        assert not o[sum(new):].any()


def test_no_sequences_and_no_tokens():
    q, kp, vp, table, cu, kv, sink, ks, vs = _cache([20], [3], 2, 1, 64, 16, seed=15)
    append, attend = _ops()
    k = torch.randn(3, 1, 64, device="cuda").to(BF)
    was = kp.clone()
    none = (table[:0], _i32([0]), kv[:0])
    assert not append(q, k, k, kp, vp, *none).any() and not attend(q, kp, vp, *none, sink).any()
    assert append(q[:0], k[:0], k[:0], kp, vp, table, _i32([0, 0]), kv).shape == (0, 2, 64)
    assert attend(q[:0], kp, vp, table, _i32([0, 0]), kv, sink).shape == (0, 2, 64)
    assert torch.equal(kp.nan_to_num(9.0), was.nan_to_num(9.0))


def test_bad_pages_are_not_followed():
    """A page number out of range where a sequence holds keys: its outputs are NaN, others' are not."""
    for new, kv in (([1, 1], [500, 70]), ([90, 1], [300, 300]), ([1, 1], [9000, 100])):
        q, kp, vp, table, cu, kvl, sink, ks, vs = _cache(kv, new, 4, 2, 64, 16, seed=9)
        for bad in (-1, kp.shape[0], -(1 << 31), (1 << 31) - 1):
            broken = table.clone()
            broken[0, 1] = bad
            o = _ops()[1](q, kp, vp, broken, cu, kvl, sink, n=16, c=8.0)
            assert torch.isnan(o[:new[0]]).all() and torch.isfinite(o[new[0]:]).all(), (new, bad)


def test_storage_order_strides_and_shared_pages():
    new, kv = [1, 40, 3], [100, 90, 33]
    a = _cache(kv, new, 8, 2, 64, 32, seed=10)
    b = _cache(kv, new, 8, 2, 64, 32, seed=10, transposed=True)
    assert b[1].stride() != a[1].stride()
    one, two = _check(a, new), _check(b, new)
    assert torch.equal(one, two)
    # Queries as a slice of a projection, tables and lengths as slices of longer rows.
    q, kp, vp, table, cu, kvl, sink, ks, vs = a
    proj = torch.randn(q.shape[0], 3, 8, 64, device="cuda").to(BF)
    proj[:, 1] = q
    wide = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    assert torch.equal(_ops()[1](proj[:, 1], kp, vp, wide[:, 2:2 + table.shape[1]], cu, kvl, sink, n=16, c=8.0), one)
    # Heads before pages in storage.
    kh, vh = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (kp, vp))
    assert kh.stride(1) > kh.stride(0)
    assert torch.equal(_ops()[1](q, kh, vh, table, cu, kvl, sink, n=16, c=8.0), one)
    # Two sequences over the same pages.
    o = _ops()[1](q[:2], kp, vp, table[[0, 0]], _i32([0, 1, 2]), _i32([100, 100]), sink, n=16, c=8.0)
    check({"o": o}, *_want(q[:2], [ks[0], ks[0]], [vs[0], vs[0]], [1, 1], sink, 16, 8.0))


def test_a_cache_past_32_bit_offsets():
    """5 GB of keys: the used pages lie beyond 2^31 bytes and beyond 2^32 bytes."""
    append, attend = _ops()
    page, Hkv, D = 128, 8, 128
    pages = 5 * (1 << 30) // (page * Hkv * D * 2)
    g, rn = _gen(11)
    kp, vp = (torch.empty(pages, Hkv, page, D, dtype=BF, device="cuda") for _ in range(2))
    ids = [pages - 1, pages // 2, 0, pages - 2]
    k, v = _norm(rn(400, Hkv, D)).to(BF), rn(400, Hkv, D).to(BF)
    q = _norm(rn(400, 16, D)).to(BF)
    table, cu, kv = _i32([ids]), _i32([0, 400]), _i32([400])
    qa = append(q, k, v, kp, vp, table, cu, kv)
    kn = torch.cat([kp[i].transpose(0, 1) for i in ids])[:400]
    assert torch.equal(torch.cat([vp[i].transpose(0, 1) for i in ids])[:400], v)
    sink = 0.3 * rn(16)
    o = attend(qa, kp, vp, table, cu, kv, sink, n=16, c=8.0)
    check({"o": o}, *_want(qa, [kn], [v], [400], sink, 16, 8.0))
    o = attend(qa[399:], kp, vp, table, _i32([0, 1]), kv, sink, n=16, c=8.0)
    check({"o": o}, *_want(qa[399:], [kn], [v], [1], sink, 16, 8.0))


def test_many_sequences():
    """Several steps of the search for a workgroup's sequence (64, 4096 and more entries)."""
    append, attend = _ops()
    for S in (63, 64, 65, 4097):
        g, rn = _gen(S)
        kv = [1 + (7 * i) % 19 for i in range(S)]
        case = _cache(kv[:65], [1] * min(S, 65), 2, 1, 64, 16, seed=S)
        q, kp, vp, table, cu, kvl, sink, ks, vs = case
        if S > 65:  # the same 65 sequences again and again
            pick = [i % 65 for i in range(S)]
            o = attend(q[pick], kp, vp, table[pick], _i32(list(range(S + 1))), kvl[pick], sink, n=16, c=8.0)
            check({"o": o[:65]}, *_want(q, ks, vs, [1] * 65, sink, 16, 8.0))
            assert torch.equal(o, o[:65][pick])
        else:
            _check(case, [1] * S)


def test_far_more_sequences_than_tokens():
    """300000 sequences of which three have a new token."""
    append, attend = _ops()
    S, at = 300000, (5, 150000, 299999)
    q, kp, vp, table, cu, kv, sink, ks, vs = _cache([700, 40, 1], [1, 1, 1], 2, 1, 64, 16, seed=16)
    lens, wide, starts = torch.zeros(S, dtype=torch.int32), torch.zeros(S, table.shape[1], dtype=torch.int32), torch.zeros(S + 1, dtype=torch.int32)
    for i, s in enumerate(at):
        lens[s], wide[s] = kv[i], table[i].cpu()
        starts[s + 1:] += 1
    o = attend(q, kp, vp, wide.cuda(), starts.cuda(), lens.cuda(), sink, n=16, c=8.0)
    check({"o": o}, *_want(q, ks, vs, [1, 1, 1], sink, 16, 8.0))
    k, v = torch.ones(3, 1, 64, dtype=BF, device="cuda"), torch.ones(3, 1, 64, dtype=BF, device="cuda")
    append(q, k, v, kp, vp, wide.cuda(), starts.cuda(), lens.cuda())
    for i, n in enumerate((700, 40, 1)):
        assert (vp[table[i, (n - 1) // 16], 0, (n - 1) % 16] == 1).all()


def test_captured_steps_follow_the_lengths():
    """Append and attention captured once; replayed as the sequences grow by a token, between eager
    calls on other inputs."""
    append, attend = _ops()
    q, kp, vp, table, cu, kv, sink, ks, vs = _cache([30, 200, 47], [1, 1, 1], 4, 2, 64, 16, seed=12, width=20)
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20)
    kp, vp = (torch.randn(60, 2, 16, 64, device="cuda").to(BF) for _ in range(2))
    k, v = torch.randn(3, 2, 64, device="cuda").to(BF), torch.randn(3, 2, 64, device="cuda").to(BF)

    def step():
        return attend(append(q, k, v, kp, vp, table, cu, kv), kp, vp, table, cu, kv, sink, n=16, c=8.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    torch.cuda.synchronize()
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        kv += 1
        want, wk, wv = step(), kp.clone(), vp.clone()
        kp[:, :, 0] += 1  # replays write and read what the eager step did
        vp[:, :, 0] += 1
        kp.copy_(wk), vp.copy_(wv)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kp, wk) and torch.equal(vp, wv), i


def test_repeats_and_other_streams():
    case = _cache([5000, 31], [1, 1], 8, 2, 128, 16, seed=13)
    args = case[:7]
    first = _ops()[1](*args, n=16, c=8.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [_ops()[1](*args, n=16, c=8.0) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        assert torch.equal(o, first)


# --- append ----------------------------------------------------------------------------------

def _tables(rows, half):
    w = 0.5 * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = 2 * torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * torch.atan(w)
    return angle.cos().float(), angle.sin().float()


def _turned(x, gain, cos, sin, pos):
    """rot(x / rms(x) gain) in float64, and the bound on its one rounding (and f32 arithmetic)."""
    x = x.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
    if gain is not None:
        y = y * gain.double()
    if cos is not None:
        a, b = y.chunk(2, -1)
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        mag = torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)
        y = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        mag = y.abs()
    return y, U * y.abs() + 1e-5 * mag


@pytest.mark.parametrize("H,Hkv,D,page", [(4, 2, 64, 16), (3, 1, 128, 48), (16, 16, 128, 64), (40, 8, 64, 32)])
@pytest.mark.parametrize("gain", [True, False])
@pytest.mark.parametrize("rotate", [True, False])
def test_append(H, Hkv, D, page, gain, rotate):
    new, kv, tail = [1, 70, 0, 5, 1], [40, 70, 9, 130, 1], 3
    g, rn = _gen(D + page)
    N = sum(new) + tail
    q, k, v = ((2 * rn(N, h, D)).to(BF) for h in (H, Hkv, Hkv))
    width = 10
    table = torch.randperm(5 * width, generator=g, device="cuda").to(torch.int32).view(5, width)
    kp, vp = (torch.full((5 * width, Hkv, page, D), 7.0, dtype=BF, device="cuda") for _ in range(2))
    cos, sin = _tables(width * page, D // 2) if rotate else (None, None)
    gq, gk = (1 + 0.2 * rn(D) for _ in range(2)) if gain else (None, None)
    print(f"[append] H{H}/{Hkv} D{D} page {page} gain {gain} rotate {rotate}", flush=True)
    qo = _ops()[0](q, k, v, kp, vp, table, _i32(_starts(new)), _i32(kv), gq, gk, cos, sin)
    torch.cuda.synchronize()
    pos = torch.tensor([kv[s] - new[s] + t for s in range(5) for t in range(new[s])], device="cuda")
    seq = torch.tensor([s for s in range(5) for _ in range(new[s])], device="cuda")
    m = sum(new)
    y, tol = _turned(q[:m], gq, cos, sin, pos)
    check({"q": qo[:m]}, {"q": y}, {"q": tol})
    assert not qo[m:].any()
    at = table.long()[seq, pos // page]
    y, tol = _turned(k[:m], gk, cos, sin, pos)
    check({"k": kp[at, :, pos % page]}, {"k": y}, {"k": tol})
    assert torch.equal(vp[at, :, pos % page], v[:m])
    # Nothing else is written.
    kp[at, :, pos % page] = 7.0
    vp[at, :, pos % page] = 7.0
    assert (kp == 7.0).all() and (vp == 7.0).all()


def test_append_out_of_range_places():
    """Positions before 0 and past the table, and bad page numbers, are not written."""
    D, page = 64, 16
    g, rn = _gen(2)
    q, k, v = (rn(6, h, D).to(BF) for h in (2, 1, 1))
    kp, vp = (torch.full((4, 1, page, D), 7.0, dtype=BF, device="cuda") for _ in range(2))
    qo = _ops()[0](q, k, v, kp, vp, _i32([[0, 1], [2, 3], [-1, 4]]), _i32([0, 2, 4, 6]), _i32([1, 33, 17]))
    assert not qo[0].any() and qo[1].any() and qo[2].any() and not qo[3].any() and qo[4:].any(dim=(1, 2)).all()
    assert torch.equal(vp[0, :, 0], v[1]) and torch.equal(vp[3, :, 15], v[2])
    vp[0, :, 0] = vp[3, :, 15] = kp[0, :, 0] = kp[3, :, 15] = 7.0
    assert (kp == 7.0).all() and (vp == 7.0).all()


def test_append_strided_projection_and_transposed_pages():
    H, Hkv, D, page, N = 4, 2, 128, 16, 20
    g, rn = _gen(3)
    proj = rn(N, (H + 2 * Hkv) * D).to(BF)
    q, k, v = (t.unflatten(1, (-1, D)) for t in proj.split([H * D, Hkv * D, Hkv * D], 1))
    table, cu, kv = _i32([[1, 0]]), _i32([0, N]), _i32([N])
    a = [torch.zeros(2, Hkv, page, D, dtype=BF, device="cuda") for _ in range(2)]
    b = [torch.zeros(2, page, Hkv, D, dtype=BF, device="cuda").transpose(1, 2) for _ in range(2)]
    one = _ops()[0](q.contiguous(), k.contiguous(), v.contiguous(), *a, table, cu, kv)
    two = _ops()[0](q, k, v, *b, table, cu, kv)
    assert torch.equal(one, two) and all(torch.equal(x, y) for x, y in zip(a, b))


# --- together --------------------------------------------------------------------------------

def test_a_block_served_in_steps_matches_the_packed_prompt():
    """One layer (residual norm, projections, append, attention, output projection) over two
    sequences: the whole prompts at once in packed attention, against the same tokens served as a
    chunk, then single tokens, through the cache. The served attention is held to its own float64
    statement elsewhere; here both paths' attention outputs lie within twice that bound."""
    from algebraic_amd.kernels.norm import add_rms_norm
    from algebraic_amd.kernels.packed import packed_flash_attention
    append, attend = _ops()
    H, Hkv, D, page, lens = 4, 2, 64, 16, [70, 33]
    d = H * D
    g, rn = _gen(20)
    x, r = rn(sum(lens), d).to(BF), rn(sum(lens), d).to(BF)
    w = (rn(d, (H + 2 * Hkv) * D) / math.sqrt(d)).to(BF)
    gain, gq, gk, sink = 1 + 0.1 * rn(d), 1 + 0.1 * rn(D), 1 + 0.1 * rn(D), 0.3 * rn(H)
    cos, sin = _tables(8 * page, D // 2)
    table = torch.randperm(16, generator=g, device="cuda").to(torch.int32).view(2, 8)
    split = [H * D, Hkv * D, Hkv * D]

    def pages():
        return [torch.zeros(16, Hkv, page, D, dtype=BF, device="cuda") for _ in range(2)]

    def project(rows):
        y, _ = add_rms_norm(x[rows], r[rows], gain)
        return [t.unflatten(1, (-1, D)) for t in (y @ w).split(split, 1)]

    cu = _starts(lens)
    q, k, v = project(slice(None))
    whole = pages()
    qr = append(q, k, v, *whole, table, _i32(cu), _i32(lens), gq, gk, cos, sin)
    kr, vr = (torch.cat([t[table[s].long()].transpose(1, 2).flatten(0, 1)[:n] for s, n in enumerate(lens)]) for t in whole)
    full = packed_flash_attention(qr, kr, vr, _i32(cu), sink, n=16, c=8.0)
    val, tol = packed_ref(qr, kr, vr, cu, sink, n=16, c=8.0)
    check({"o": full}, val, tol, "packed")
    steps = pages()
    done = [0, 0]
    for new in ([64, 20], [1, 10], [1, 1], [4, 2]):
        rows = [i for s, m in enumerate(new) for i in range(cu[s] + done[s], cu[s] + done[s] + m)]
        done = [a + b for a, b in zip(done, new)]
        q, k, v = project(rows)
        args = (table, _i32(_starts(new)), _i32(done))
        qs = append(q, k, v, *steps, *args, gq, gk, cos, sin)
        o = attend(qs, *steps, *args, sink, n=16, c=8.0)
        # The projections of other row counts may round otherwise; the attention is compared on
        # what each path put in.
        for s, m in enumerate(new):
            at = slice(_starts(new)[s], _starts(new)[s] + m)
            ks, vs = (t[table[s].long()].transpose(1, 2).flatten(0, 1)[:done[s]] for t in steps)
            check({"o": o[at]}, *_want(qs[at], [ks], [vs], [m], sink, 16, 8.0), f"step {new} sequence {s}")
        diff = (o.double() - val["o"][rows]).abs().max() / val["o"].abs().max()
        assert diff < 0.05, diff
    assert done == lens

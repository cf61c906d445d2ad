"""GPU: calls of the packed, paged and residual-norm operators at the edges of what they take, against
the float64 statement of tests/packed_ref.py."""

import math

import pytest

from packed_ref import check, head_ref, packed_ref

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
    return lambda *s: torch.randn(*s, device="cuda", generator=g)


def _norm(t):
    return t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()


def _held(S, width, page, new, H, Hkv, D, seed):
    """Queries, a cache whose every place is filled, its table, and each sequence's keys and values."""
    rn = _gen(seed)
    kp, vp = _norm(rn(S * width, Hkv, page, D)).to(BF), rn(S * width, Hkv, page, D).to(BF)
    table = rn(S * width).argsort().to(torch.int32).view(S, width)
    rows = lambda t, s: t[table[s].long()].transpose(1, 2).flatten(0, 1)  # noqa: E731
    q = _norm(rn(sum(new), H, D)).to(BF)
    return q, kp, vp, table, 0.3 * rn(H), [rows(kp, s) for s in range(S)], [rows(vp, s) for s in range(S)]


def _row(q, k, v, sink, pos, n=16, c=8.0):
    """One sequence's tokens at `pos` over its keys: value and bound."""
    val, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    G = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        s = None if sink is None else sink[h].double()
        hv, ht = head_ref(q[:, h].double(), k[:, h // G].double(), v[:, h // G].double(), s, n=n, c=c, positions=pos)
        val[:, h], tol[:, h] = hv["o"], ht["o"]
    return {"o": val}, {"o": tol}


# A sequence that outgrew its row of the table by `past` positions; another one beside it.
@pytest.mark.parametrize("new,width,past,H,Hkv", [
    ([2, 1], 2, 1, 4, 2), ([3, 1], 2, 2, 4, 4), ([1, 1], 3, 1, 4, 2), ([40, 1], 4, 39, 4, 1),
    ([150, 3], 10, 40, 4, 2), ([150, 3], 11, 150, 4, 2), ([2], 562, 1, 4, 1), ([200], 375, 50, 2, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sink", [False, True])
def test_lengths_past_the_table(new, width, past, H, Hkv, D, sink):
    """Tokens stand where kv_lens puts them: those that the table reaches see every key up to their
    own, those behind it are NaN, and other sequences are as they were."""
    page, reach = 16, 16 * width
    print(f"[edges] {new} tokens, {past} past {reach} positions, H{H}/{Hkv} D{D} sink {sink}", flush=True)
    q, kp, vp, table, s, ks, vs = _held(len(new), width, page, new, H, Hkv, D, seed=sum(new) + D)
    s = s if sink else None
    kv = [reach + past] + [reach - 1] * (len(new) - 1)
    o = _ops()[1](q, kp, vp, table, _i32(_starts(new)), _i32(kv), s, n=16, c=8.0)
    torch.cuda.synchronize()
    inside = new[0] - past
    assert torch.isnan(o[inside:new[0]]).all()
    if inside:
        check({"o": o[:inside]}, *_row(q[:inside], ks[0], vs[0], s, torch.arange(reach - inside, reach, device="cuda")), "inside")
    for i in range(1, len(new)):
        at = slice(_starts(new)[i], _starts(new)[i + 1])
        check({"o": o[at]}, *_row(q[at], ks[i][:kv[i]], vs[i][:kv[i]], s, torch.arange(kv[i] - new[i], kv[i], device="cuda")), "beside")


def test_lengths_at_the_largest_number():
    for new in ([1, 1], [150, 3]):
        q, kp, vp, table, s, ks, vs = _held(2, 12, 16, new, 4, 2, 64, seed=1)
        o = _ops()[1](q, kp, vp, table, _i32(_starts(new)), _i32([(1 << 31) - 1, 20]), s, n=16, c=8.0)
        assert torch.isnan(o[:new[0]]).all() and torch.isfinite(o[new[0]:]).all()


@pytest.mark.parametrize("new,width", [([1, 1], 4), ([1, 1], 2000), ([1], 8192), ([2, 1], 40), ([60, 40], 4), ([150], 400)],
                         ids=["whole", "ranges", "many-ranges", "two", "chunks", "chunk-in-ranges"])
@pytest.mark.parametrize("G", [1, 4])
def test_a_switched_off_sink_and_rows_without_keys(new, width, G):
    """A head whose sink is -inf has none: a row that holds no key is zeros there as elsewhere, and
    other rows are what they are without the sink."""
    H, D = 2 * G, 64
    q, kp, vp, table, s, ks, vs = _held(len(new), width, 16, new, H, 2, D, seed=width + G)
    s[0] = s[-1] = -math.inf
    cu = _i32(_starts(new))
    o = _ops()[1](q, kp, vp, table, cu, _i32([0] * len(new)), s, n=16, c=8.0)
    assert torch.equal(o, torch.zeros_like(o)), (new, width)
    kv = [new[0] // 2] + [50] * (len(new) - 1)  # the first sequence's earlier tokens lie before position 0
    o = _ops()[1](q, kp, vp, table, cu, _i32(kv), s, n=16, c=8.0)
    gone = new[0] - kv[0]
    assert torch.equal(o[:gone], torch.zeros_like(o[:gone]))
    for i in range(len(new)):
        a, b = _starts(new)[i] + (gone if i == 0 else 0), _starts(new)[i + 1]
        if a < b:
            pos = torch.arange(kv[i] - (b - a), kv[i], device="cuda")
            check({"o": o[a:b]}, *_row(q[a:b], ks[i][:kv[i]], vs[i][:kv[i]], s, pos))


@pytest.mark.parametrize("lens,H,Hkv,D", [([70, 1], 4, 2, 64), ([1500], 3, 1, 128)])
def test_a_switched_off_sink_in_packed_rows(lens, H, Hkv, D):
    from algebraic_amd.kernels.packed import packed_flash_attention
    rn = _gen(H)
    N, cu = sum(lens), _starts(lens)
    for scale in (1.0, 40.0):  # both forms of the weights
        leaves = [t.to(BF).requires_grad_(True) for t in (_norm(rn(N, H, D)) * scale, _norm(rn(N, Hkv, D)), rn(N, Hkv, D))]
        do, s = rn(N, H, D).to(BF), 0.3 * rn(H)
        s[0] = -math.inf
        s.requires_grad_(True)
        o = packed_flash_attention(*leaves, _i32(cu), s, n=16, c=8.0)
        got = dict(zip(("o", "dq", "dk", "dv", "dsink"), (o, *torch.autograd.grad(o, [*leaves, s], do))))
        check(got, *packed_ref(*leaves, cu, s, do, n=16, c=8.0))


# --- single tokens ---------------------------------------------------------------------------

def _awkward(t):
    """(1, heads, D) views of `t`'s values whose token stride means nothing: one element, and more
    than 32-bit offsets reach."""
    _, h, D = t.shape
    one = t.reshape(h, D, 1).permute(2, 0, 1)
    wide = torch.as_strided(t.contiguous(), (1, h, D), (1 << 28, D, 1))
    odd = torch.as_strided(t.contiguous(), (1, h, D), (h * D + 4, D, 1))
    assert one.stride(0) == 1 and torch.equal(one, t)
    return one, wide, odd


def test_one_token_of_any_token_stride():
    from algebraic_amd.kernels.packed import packed_flash_attention
    rn = _gen(5)
    H, Hkv, D = 4, 2, 64
    q, k, v, do = (rn(1, h, D).to(BF) for h in (H, Hkv, Hkv, H))
    cu = _i32([0, 1])

    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = packed_flash_attention(*leaves, cu, n=16, c=8.0)
        return [o, *torch.autograd.grad(o, leaves, do)]

    kp, vp = (rn(4, Hkv, 16, D).to(BF) for _ in range(2))
    table, kv = _i32([[2, 1]]), _i32([20])
    want, rows = run(q, k, v, do), _ops()[1](q, kp, vp, table, cu, kv, n=16, c=8.0)
    wk, wv = kp.clone(), vp.clone()
    wq = _ops()[0](q, k, v, wk, wv, table, cu, kv)
    for qa, ka, va, da in zip(*(_awkward(t) for t in (q, k, v, do))):
        print(f"[edges] one token, strides {qa.stride()}", flush=True)
        for a, b in zip(run(qa, ka, va, da), want):
            assert torch.equal(a, b)
        assert torch.equal(_ops()[1](qa, kp, vp, table, cu, kv, n=16, c=8.0), rows)
        ck, cv = kp.clone(), vp.clone()
        assert torch.equal(_ops()[0](qa, ka, va, ck, cv, table, cu, kv), wq)
        assert torch.equal(ck, wk) and torch.equal(cv, wv)


def test_one_page_and_one_head_of_any_stride():
    """The strides of axes of length one are never used, and not looked at."""
    rn = _gen(6)
    q, k = rn(3, 2, 64).to(BF), rn(3, 1, 64).to(BF)
    kp, vp = (rn(1, 1, 16, 64).to(BF) for _ in range(2))
    args = (_i32([[0]]), _i32([0, 3]), _i32([13]))
    want = _ops()[1](q, kp, vp, *args, n=16, c=8.0)
    odd = [torch.as_strided(t, t.shape, (1, 4, 64, 1)) for t in (kp, vp)]
    assert torch.equal(_ops()[1](q, *odd, *args, n=16, c=8.0), want)
    other = [t.clone() for t in (kp, vp)]
    _ops()[0](q, k, k, *other, *args)
    _ops()[0](q, k, k, *odd, *args)
    assert torch.equal(kp, other[0]) and torch.equal(vp, other[1])


# --- gradients -------------------------------------------------------------------------------

def test_second_derivatives_are_refused():
    """The backward passes are kernels without one of their own: a penalty on their results raises,
    and does not drop its terms, whether or not the cotangent has a gradient."""
    from algebraic_amd.kernels.norm import add_rms_norm
    from algebraic_amd.kernels.packed import packed_flash_attention
    rn = _gen(7)
    q, k, v = (rn(5, h, 64).to(BF).requires_grad_(True) for h in (2, 1, 1))
    s, gain = rn(2).requires_grad_(True), rn(64).requires_grad_(True)
    x, r = (rn(5, 64).to(BF).requires_grad_(True) for _ in range(2))
    for call, leaves in ((lambda: packed_flash_attention(q, k, v, _i32([0, 5]), s), (q, k, v, s)),
                         (lambda: add_rms_norm(x, r, gain)[0], (x, r, gain))):
        for loss in (lambda o: o.float().square().sum(), lambda o: o.sum()):
            once = torch.autograd.grad(loss(call()), leaves)
            grads = torch.autograd.grad(loss(call()), leaves, create_graph=True)
            for leaf, a, b in zip(leaves, once, grads):
                assert torch.equal(a, b.detach())
                with pytest.raises(RuntimeError, match="no second derivative"):
                    torch.autograd.grad(b.float().square().sum() + leaf.float().square().sum(), leaf, retain_graph=True)
    # The stream's own gradient is what came in, differentiable as ever.
    y, h = add_rms_norm(x, r, gain)
    (g,) = torch.autograd.grad(h.float().square().sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(g.float().sum(), x)
    assert torch.equal(gg, torch.full_like(gg, 2.0))


# --- gradients of scores out of range --------------------------------------------------------

def _backward_of_weights(q, k, v, sink, do, n, c):
    """One head in float64 (all rows of one sequence) and bounds that hold no rounding of o: P and dS are
    rounded to bf16 for their products and the results to bf16, u = 2^-8 each; di = sum_j P dP, like
    every other sum, is f32, whose share is 1e-4 of the magnitudes added up (16 times a weight's few
    2^-24, and up to 1500 terms' 2^-24 each)."""
    U, F = 2.0 ** -8, 1e-4
    alpha = 1.0 / (math.sqrt(q.shape[1]) * c)
    x = (q @ k.T) * alpha
    dead = torch.ones_like(x, dtype=torch.bool).triu(1)
    a = (n * torch.asinh(x)).masked_fill(dead, -math.inf)
    ab = torch.full_like(a[:, :1], -math.inf) if sink is None else (n * torch.asinh(sink / c)).expand(a.shape[0], 1)
    both = torch.softmax(torch.cat([a, ab], 1), 1)
    p, pb = both[:, :-1], both[:, -1:]
    dp, mag_dp = do @ v.T, do.abs() @ v.abs().T
    di, mag_di = (p * dp).sum(1, keepdim=True), (p * mag_dp).sum(1, keepdim=True)
    f = n * alpha * p / torch.sqrt(1 + x * x)
    ds = f * (dp - di)
    off = U * ds.abs() + F * f * (mag_dp + mag_di)
    val = {"dq": ds @ k, "dk": ds.T @ q, "dv": p.T @ do}
    tol = {"dq": off @ k.abs(), "dk": off.T @ q.abs(), "dv": (U + F) * (p.T @ do.abs())}
    tol = {m: t + U * val[m].abs() for m, t in tol.items()}
    if sink is not None:
        rb = n / torch.sqrt(1 + (sink / c) ** 2) / c
        val["dsink"], tol["dsink"] = -(pb * di).sum() * rb, F * (pb * mag_di).sum() * rb
    return val, tol


@pytest.mark.parametrize("lens,H,Hkv,D", [([300, 70], 2, 2, 64), ([513, 1, 40], 4, 1, 128), ([1500], 3, 1, 128)],
                         ids=["heads", "group", "ranges"])
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("n", [16, 64])
def test_gradients_of_scores_out_of_range_do_not_see_the_output_rounded(lens, H, Hkv, D, sink, n):
    """Values that share a large part: dP and di are far larger than their difference, and a di of the
    rounded output would be off by more than that. As flash_attention's range guard computes it."""
    from algebraic_amd.kernels.packed import packed_flash_attention
    rn = _gen(D + H)
    N, cu, G = sum(lens), _starts(lens), H // Hkv
    q, k = _norm(rn(N, H, D)), _norm(rn(N, Hkv, D))
    q[..., 0], k[..., 0] = 1600.0, 8.0  # every score near 200 (141 at D = 128)
    leaves = [t.to(BF).requires_grad_(True) for t in (q, k, 3 + 0.1 * rn(N, Hkv, D))]
    do, s = (1 + rn(N, H, D)).to(BF), (1600.0 + 30 * rn(H)).requires_grad_(True) if sink else None
    print(f"[edges] far scores {lens} H{H}/{Hkv} D{D} sink {sink} n {n}", flush=True)
    o = packed_flash_attention(*leaves, _i32(cu), s, n=n, c=8.0)
    got = dict(zip(("dq", "dk", "dv", "dsink"), torch.autograd.grad(o, [*leaves] + ([s] if sink else []), do)))
    val = {m: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for m, t in got.items()}
    tol = {m: torch.zeros_like(t) for m, t in val.items()}
    for a, b in zip(cu, cu[1:]):
        for h in range(H):
            hv, ht = _backward_of_weights(*(t[a:b, i].detach().double() for t, i in zip(leaves, (h, h // G, h // G))),
                                          s[h].detach().double() if sink else None, do[a:b, h].double(), n, 8.0)
            for m in hv:
                at = (h,) if m == "dsink" else (slice(a, b), h if m == "dq" else h // G)
                val[m][at] += hv[m]
                tol[m][at] += ht[m]
    check(got, val, tol)


# --- the 8-bit norm --------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 512, 4096])
@pytest.mark.parametrize("gain", [False, True])
def test_eight_bits_are_the_quotient_of_the_stored_scale(d, gain):
    """y8 = e4m3(y / scale), scale = max|y| / 448, to the bit: whole numbers, whose squares add up
    without a rounding in any order, and a power-of-two width leave the norm one value."""
    from algebraic_amd.kernels.norm import add_rms_norm_fp8
    rn = _gen(d)
    x, r = ((3 * rn(700, d)).round().to(BF) for _ in range(2))
    g = (1 + 0.2 * rn(d)) if gain else None
    y8, scale, s = add_rms_norm_fp8(x, r, g)
    h = s.cpu().double()
    assert torch.equal(h, (x.double() + r.double()).cpu())
    # f32 arithmetic, every step rounded once: the mean square is exact before eps.
    f32 = lambda t: t.float().double()  # noqa: E731
    ms = f32(f32((h * h).mean(-1, keepdim=True)) + float(torch.tensor(1e-5)))
    tau = f32(1.0 / f32(ms.sqrt()))
    y = f32(h * tau)
    if gain:
        y = f32(y * g.cpu().double())
    want = f32(y.abs().amax(-1, keepdim=True) / 448.0)
    assert torch.equal(scale.cpu().double(), want)
    assert torch.equal(y8.cpu().float(), f32(y / want).float().clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float())


# --- more than 64 sequences in ranges --------------------------------------------------------

def _cached(kv, new, H, Hkv, D, seed):
    """As _held, with kv_lens `kv`; and whether the call runs over ranges of keys."""
    from algebraic_amd import _lib
    width = -(-max(kv) // 16)
    q, kp, vp, table, s, ks, vs = _held(len(kv), width, 16, new, H, Hkv, D, seed)
    ranges = _lib.load().alg_paged_attn_workspace_size(sum(new), len(kv), H, Hkv, D, width, 16) > 0
    want = {"o": torch.zeros(q.shape, dtype=torch.float64, device="cuda")}
    tol = {"o": torch.zeros_like(want["o"])}
    for i, m in enumerate(new):
        at = slice(_starts(new)[i], _starts(new)[i + 1])
        v, t = _row(q[at], ks[i][:kv[i]], vs[i][:kv[i]], s, torch.arange(kv[i] - m, kv[i], device="cuda"))
        want["o"][at], tol["o"][at] = v["o"], t["o"]
    return (q, kp, vp, table, _i32(_starts(new)), _i32(kv), s), ranges, want, tol


@pytest.mark.parametrize("S", [65, 100])
def test_single_tokens_of_many_sequences_in_ranges(S):
    kv = [1000 + (811 * i) % 2000 for i in range(S)]
    kv[3] = 1  # ranges without a key
    args, ranges, want, tol = _cached(kv, [1] * S, 2, 1, 64, seed=S)
    assert ranges
    print(f"[edges] {S} single tokens in ranges", flush=True)
    check({"o": _ops()[1](*args, n=16, c=8.0)}, want, tol)


@pytest.mark.parametrize("S,H,Hkv,D", [(66, 2, 1, 64), (70, 2, 1, 128)])
def test_chunks_of_many_sequences_in_ranges(S, H, Hkv, D):
    new = [40 + i % 11 for i in range(S)]
    kv = [300 + (277 * i) % 1200 for i in range(S)]
    kv[5] = new[5]
    args, ranges, want, tol = _cached(kv, new, H, Hkv, D, seed=S)
    assert ranges
    print(f"[edges] {S} chunks in ranges", flush=True)
    check({"o": _ops()[1](*args, n=16, c=8.0)}, want, tol)


@pytest.mark.parametrize("sink", [False, True])
def test_packed_sequences_in_ranges_past_64(sink):
    from algebraic_amd import _lib
    from algebraic_amd.kernels.packed import packed_flash_attention
    H, Hkv, D = 16, 1, 64
    lens = [50 + (13 * i) % 21 for i in range(66)]
    N, cu = sum(lens) + 9, _starts(lens)
    base = _lib.load().alg_packed_attn_bwd_workspace_size(N, N, H, Hkv, D)  # short ones: no ranges, more slots
    assert _lib.load().alg_packed_attn_bwd_workspace_size(N, 66, H, Hkv, D) >= base + 2 * N * Hkv * D * 4
    rn = _gen(66)
    leaves = [t.to(BF).requires_grad_(True) for t in (_norm(rn(N, H, D)), _norm(rn(N, Hkv, D)), rn(N, Hkv, D))]
    do, s = rn(N, H, D).to(BF), (0.3 * rn(H)).requires_grad_(True) if sink else None
    print("[edges] 66 packed sequences in ranges", flush=True)
    o = packed_flash_attention(*leaves, _i32(cu), s, n=16, c=8.0)
    wrt = [*leaves] + ([s] if sink else [])
    got = dict(zip(("o", "dq", "dk", "dv", "dsink"), (o, *torch.autograd.grad(o, wrt, do))))
    for name in ("o", "dq", "dk", "dv"):
        assert not got[name][-9:].any(), name
    check(got, *packed_ref(*leaves, cu, s, do, n=16, c=8.0))


# --- captured steps --------------------------------------------------------------------------

def test_captured_steps_write_the_cache_themselves():
    """Append and attention captured once; before each replay the new tokens' places hold something
    else than the eager step wrote there."""
    append, attend = _ops()
    rn = _gen(8)
    table = rn(60).argsort().to(torch.int32).view(3, 20)
    kp, vp = (rn(60, 2, 16, 64).to(BF) for _ in range(2))
    q, k, v = rn(3, 4, 64).to(BF), rn(3, 2, 64).to(BF), rn(3, 2, 64).to(BF)
    cu, kv, s = _i32([0, 1, 2, 3]), _i32([30, 200, 47]), 0.3 * rn(4)

    def step():
        return attend(append(q, k, v, kp, vp, table, cu, kv), kp, vp, table, cu, kv, s, n=16, c=8.0)

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
            t.copy_(rn(*t.shape))
        kv += 1
        before = kp.clone(), vp.clone()
        want, wk, wv = step(), kp.clone(), vp.clone()
        assert not torch.equal(wk, before[0]) and not torch.equal(wv, before[1])
        kp.copy_(before[0]), vp.copy_(before[1])
        torch.cuda.synchronize()
        print(f"[edges] replay {i}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kp, wk) and torch.equal(vp, wv), i


def test_a_captured_call_over_ranges_follows_the_lengths():
    """One captured call over ranges of keys, replayed with other lengths between eager ones: ranges
    that were written become empty and the other way round."""
    attend = _ops()[1]
    rn = _gen(9)
    q, kp, vp, table, s, _, _ = _held(2, 400, 16, [1, 1], 8, 2, 128, seed=9)
    cu, kv = _i32([0, 1, 2]), _i32([6400, 6400])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(q, kp, vp, table, cu, kv, s, n=16, c=8.0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(q, kp, vp, table, cu, kv, s, n=16, c=8.0)
    torch.cuda.synchronize()
    for lens in ([6400, 6400], [1, 6000], [700, 0], [6399, 257], [0, 0]):
        q.copy_(_norm(rn(*q.shape)))
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        want = attend(q, kp, vp, table, cu, kv, s, n=16, c=8.0)
        torch.cuda.synchronize()
        print(f"[edges] replay of {lens}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(out).all(), lens

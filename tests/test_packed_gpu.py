"""GPU: attention over packed sequences with grouped heads, forward and backward, element by element
against the float64 statement of tests/packed_ref.py within bounds derived there."""

import pytest

from packed_ref import check, packed_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _op():
    from algebraic_amd.kernels.packed import packed_flash_attention
    return packed_flash_attention


def _inputs(lens, H, Hkv, D, *, tail=0, sink="heads", scale=1.0, shift=0.0, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    N = sum(lens) + tail
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    nrm = lambda t: t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()  # noqa: E731
    bf = torch.bfloat16
    q, k, v, do = nrm(rn(N, H, D)) * scale, nrm(rn(N, Hkv, D)), rn(N, Hkv, D), rn(N, H, D)
    if shift:  # every score of a row moved the same way: q and k share a direction
        q[..., 0], k[..., 0] = shift, 8.0
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    s = {"none": None, "one": 0.3 * rn(1), "heads": 0.3 * rn(H)}[sink]
    leaves = [t.to(bf).requires_grad_(True) for t in (q, k, v)]
    return leaves, None if s is None else s.requires_grad_(True), do.to(bf), cu


def _run(leaves, sink, do, cu, n, c):
    o = _op()(*leaves, torch.tensor(cu, dtype=torch.int32, device="cuda"), sink, n=n, c=c)
    grads = torch.autograd.grad(o, [*leaves] + ([] if sink is None else [sink]), do)
    torch.cuda.synchronize()
    return dict(zip(("o", "dq", "dk", "dv", "dsink"), (o, *grads)))


LENS = [
    [1], [2, 1, 1], [64], [63, 65, 1], [128, 127, 129], [0, 5, 0, 0, 70, 0], [300, 17, 191], [32] * 70,
]


@pytest.mark.parametrize("lens", LENS, ids=[f"{len(x)}seq{sum(x)}" for x in LENS])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (4, 1, 128), (6, 2, 64), (3, 1, 128), (16, 2, 64)])
def test_lengths_and_groups(lens, H, Hkv, D):
    print(f"[packed] {lens[:4]} H{H}/{Hkv} D{D}", flush=True)
    leaves, sink, do, cu = _inputs(lens, H, Hkv, D, seed=H + D)
    check(_run(leaves, sink, do, cu, 16, 8.0), *packed_ref(*leaves, cu, sink, do, n=16, c=8.0))


@pytest.mark.parametrize("G,D,T", [(1, 128, 700), (5, 64, 333), (32, 128, 150), (128, 64, 65)])
def test_long_rows_and_large_groups(G, D, T):
    print(f"[packed] group {G} D{D} T{T}", flush=True)
    leaves, sink, do, cu = _inputs([T, 40], 2 * G, 2, D, seed=G)
    check(_run(leaves, sink, do, cu, 16, 8.0), *packed_ref(*leaves, cu, sink, do, n=16, c=8.0))


@pytest.mark.parametrize("S", [64, 65, 200])
def test_many_ragged_sequences(S):
    """On both sides of 64 sequences, where the workgroups' order changes; empty ones among them."""
    lens = [(37 * i) % 23 if i % 5 else 0 for i in range(S - 2)] + [150, 1]
    print(f"[packed] {S} sequences", flush=True)
    leaves, sink, do, cu = _inputs(lens, 6, 2, 64, tail=5, seed=S)
    check(_run(leaves, sink, do, cu, 16, 8.0), *packed_ref(*leaves, cu, sink, do, n=16, c=8.0))


@pytest.mark.parametrize("D", [64, 128])
def test_a_long_sequence(D):
    leaves, sink, do, cu = _inputs([2900, 130], 2, 1, D, seed=15)
    check(_run(leaves, sink, do, cu, 16, 8.0), *packed_ref(*leaves, cu, sink, do, n=16, c=8.0))


@pytest.mark.parametrize("n", [2, 4, 8, 32, 64, 1024])
@pytest.mark.parametrize("sink", ["none", "one", "heads"])
def test_exponents_and_sinks(n, sink):
    leaves, s, do, cu = _inputs([77, 130], 4, 2, 64, sink=sink, seed=n)
    c = 8.0 if n <= 64 else 400.0
    print(f"[packed] n {n} sink {sink}", flush=True)
    check(_run(leaves, s, do, cu, n, c), *packed_ref(*leaves, cu, s, do, n=n, c=c))


@pytest.mark.parametrize("scale,shift,c", [(30.0, 0.0, 8.0), (1.0, 400.0, 8.0), (1.0, -400.0, 8.0), (3.0, 0.0, 0.01),
                                           (1.0, -20.0, 8.0), (1.0, 1e4, 8.0)])
@pytest.mark.parametrize("sink", ["none", "heads"])
def test_scores_outside_the_plain_form(scale, shift, c, sink):
    """Scores far above and below the bound of the plain form, whole rows of them: the careful form,
    forward and backward; one sequence stays inside."""
    leaves, s, do, cu = _inputs([150, 90], 4, 2, 128, sink=sink, scale=scale, shift=shift, seed=5)
    with torch.no_grad():
        leaves[0][150:] = _inputs([150, 90], 4, 2, 128, seed=6)[0][0][150:] * 0.25
    print(f"[packed] scale {scale} shift {shift} c {c} sink {sink}", flush=True)
    check(_run(leaves, s, do, cu, 16, c), *packed_ref(*leaves, cu, s, do, n=16, c=c))


def _ranges(N, S, H, Hkv, D):
    """Whether the forward (and dQ), and whether dK/dV of these sizes run over ranges, by the sums
    that their workspaces hold."""
    from algebraic_amd import _lib
    lib = _lib.load()
    fwd, bwd = lib.alg_packed_attn_fwd_workspace_size(N, S, H, Hkv, D), lib.alg_packed_attn_bwd_workspace_size(N, S, H, Hkv, D)
    base = lib.alg_packed_attn_bwd_workspace_size(8, 8, H, Hkv, D)
    sums = max(bwd - base - N * H * 4 - 65536, 0)
    return fwd > 0, sums >= (2 * N * H * D * 4 if fwd else 0) + 2 * 2 * N * Hkv * D * 4


@pytest.mark.parametrize("lens,H,Hkv,D", [([1500], 3, 1, 128), ([1100, 300, 7], 4, 1, 64), ([2100, 1, 0, 900], 2, 2, 64),
                                          ([2200, 1, 0, 1700], 2, 2, 64), ([400], 16, 1, 128), ([65, 900], 12, 1, 64)])
@pytest.mark.parametrize("sink,n", [("heads", 16), ("none", 4), ("one", 64)])
def test_few_heads_in_ranges(lens, H, Hkv, D, sink, n):
    """Keys and rows split over workgroups, tokens behind the last sequence among them; one on the
    other side of the rule."""
    N = sum(lens) + 70
    assert any(_ranges(N, len(lens), H, Hkv, D)) == (lens != [2100, 1, 0, 900])
    print(f"[packed] ranges {lens} H{H}/{Hkv} D{D} sink {sink} n {n} {_ranges(N, len(lens), H, Hkv, D)}", flush=True)
    leaves, s, do, cu = _inputs(lens, H, Hkv, D, tail=70, sink=sink, seed=N)
    got = _run(leaves, s, do, cu, n, 8.0)
    for name in ("o", "dq", "dk", "dv"):
        assert not got[name][-70:].any(), name
    check(got, *packed_ref(*leaves, cu, s, do, n=n, c=8.0))
    again = _run(leaves, s, do, cu, n, 8.0)
    for name in got:
        assert torch.equal(got[name], again[name]), name


@pytest.mark.parametrize("sink", ["none", "heads", "huge"])
@pytest.mark.parametrize("late", [400.0, -400.0, -30.0])
def test_ranges_of_both_forms(sink, late):
    """A row whose first keys have ordinary scores and whose last ones lie outside the plain form (or
    the other way round): ranges of different forms are joined, and the backward knows it."""
    leaves, s, do, cu = _inputs([1500], 3, 1, 128, sink="none" if sink == "none" else "heads", seed=17)
    assert all(_ranges(1500, 1, 3, 1, 128))
    with torch.no_grad():
        leaves[0][..., 0], leaves[1][..., 0] = 8.0, 0.0
        leaves[1][700:1100, :, 0] = late
        if sink == "huge":
            s[0], s[1], s[2] = 1e3, -1e3, 300.0
    print(f"[packed] ranges of both forms, late {late} sink {sink}", flush=True)
    check(_run(leaves, s, do, cu, 16, 8.0), *packed_ref(*leaves, cu, s, do, n=16, c=8.0))


def test_ranges_that_are_not_finite_stay_alone():
    leaves, s, do, cu = _inputs([1300, 200], 3, 1, 64, seed=18)
    val, tol = packed_ref(*leaves, cu, s, do, n=16, c=8.0)
    with torch.no_grad():
        leaves[1][600] = float("nan")
        leaves[2][1290] = float("inf")
    got = _run(leaves, s, do, cu, 16, 8.0)
    assert not torch.isfinite(got["o"][600:1300]).any()
    sel = lambda d: {m: d[m][1300:] for m in ("o", "dq", "dk", "dv")}  # noqa: E731
    check(sel(got), sel(val), sel(tol))


@pytest.mark.parametrize("n,c", [(2, 0.05), (2, 0.01), (4, 0.05), (8, 0.1), (32, 8.0)])
def test_rows_of_large_scores_of_both_signs(n, c):
    """Scores up to hundreds on either side of zero in one row, down to sequences of a few keys: the
    smallest weights are far below the row's mean."""
    leaves, s, do, cu = _inputs([1, 2, 3, 5, 8, 70, 200], 2, 2, 128, sink="none", scale=20.0, seed=21)
    print(f"[packed] both signs n {n} c {c}", flush=True)
    check(_run(leaves, None, do, cu, n, c), *packed_ref(*leaves, cu, None, do, n=n, c=c))


@pytest.mark.parametrize("D", [8, 40, 96, 120])
def test_other_widths(D):
    leaves, s, do, cu = _inputs([70, 33], 4, 2, D, seed=D)
    check(_run(leaves, s, do, cu, 16, 8.0), *packed_ref(*leaves, cu, s, do, n=16, c=8.0))


def test_tokens_behind_the_last_sequence():
    leaves, s, do, cu = _inputs([60, 75], 4, 2, 64, tail=200, seed=3)
    got = _run(leaves, s, do, cu, 16, 8.0)
    for name in ("o", "dq", "dk", "dv"):
        assert not got[name][135:].any(), name
    check(got, *packed_ref(*leaves, cu, s, do, n=16, c=8.0))
    none = _run(leaves, s, do, [0], 16, 8.0)  # no sequence at all
    for name, t in none.items():
        assert not t.any(), name


def test_a_sequence_that_is_not_finite_stays_alone():
    leaves, s, do, cu = _inputs([70, 64, 40], 4, 2, 64, seed=4)
    val, tol = packed_ref(*leaves, cu, s, do, n=16, c=8.0)
    with torch.no_grad():
        for i, bad in enumerate((float("nan"), float("inf"), float("nan"))):
            leaves[i][70:134] = bad
        do[70:134] = float("nan")
    got = _run(leaves, s, do, cu, 16, 8.0)
    assert not torch.isfinite(got["o"][70:134]).any()
    keep = [*range(70), *range(134, 174)]
    sel = lambda d: {m: d[m][keep] for m in ("o", "dq", "dk", "dv")}  # noqa: E731
    check(sel(got), sel(val), sel(tol))


def test_slices_of_one_projection_and_an_expanded_cotangent():
    """q, k and v as views of one (N, (H + 2 Hkv) D) projection, read in place; head-major storage;
    a cotangent expanded over heads; gradients reach the projection."""
    H, Hkv, D, lens = 4, 2, 64, [90, 41]
    leaves, s, do, cu = _inputs(lens, H, Hkv, D, seed=8)
    proj = torch.cat([t.detach().reshape(131, -1) for t in leaves], 1).requires_grad_(True)
    q, k, v = (t.unflatten(1, (-1, D)) for t in proj.split([H * D, Hkv * D, Hkv * D], 1))
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
    o = _op()(q, k, v, cut, s, n=16, c=8.0)
    do1 = do[:, :1].expand(-1, H, -1)
    (dproj, ds) = torch.autograd.grad(o, (proj, s), do1)
    val, tol = packed_ref(*leaves, cu, s, do1, n=16, c=8.0)
    parts = dict(zip(("dq", "dk", "dv"), (t.unflatten(1, (-1, D)) for t in dproj.split([H * D, Hkv * D, Hkv * D], 1))))
    check({"o": o, **parts, "dsink": ds}, val, tol)
    head_major = [t.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True) for t in leaves]
    o2 = _op()(*head_major, cut, s, n=16, c=8.0)
    assert torch.equal(o2, o)
    got = torch.autograd.grad(o2, [*head_major, s], do1.transpose(0, 1).contiguous().transpose(0, 1))
    for a, b in zip(got, (*parts.values(), ds)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,H,Hkv", [(64, 2, 1), (128, 4, 4)])
def test_rows_past_32_bit_offsets(D, H, Hkv):
    """q, k, v and the cotangent as slices of rows of 16 MB: the later tokens lie beyond 2^31 and 2^32
    bytes."""
    lens, row = [290, 1, 30], 8 * (1 << 20)
    leaves, s, do, cu = _inputs(lens, H, Hkv, D, seed=19)
    wide = torch.empty(sum(lens), row, dtype=torch.bfloat16, device="cuda")
    views, at = [], row // 2
    for t in (*leaves, do):
        n = t[0].numel()
        views.append(wide[:, at:at + n].unflatten(1, (-1, D)).copy_(t.detach()))
        at += n
    print(f"[packed] rows of {row} elements D{D}", flush=True)
    far = [t.requires_grad_(True) for t in views[:3]]
    assert far[0].stride(0) == row
    check(_run(far, s, views[3], cu, 16, 8.0), *packed_ref(*leaves, cu, s, do, n=16, c=8.0))


def test_equal_lengths_match_flash_attention():
    """Rows of one length with a key head a query head are flash_attention's, whose own bounds
    are two roundings of its scaled queries wider: both within the float64 statement's."""
    from algebraic_amd.kernels.flash import flash_attention
    leaves, s, do, cu = _inputs([192, 192], 2, 2, 64, seed=9)
    got = _run(leaves, s, do, cu, 16, 8.0)
    b = [t.detach().unflatten(0, (2, 192)).requires_grad_(True) for t in leaves]
    o = flash_attention(*b, s, kind="asinh", n=16, c=8.0, block=192, range_guard=True, layout="bthd")
    grads = torch.autograd.grad(o, [*b, s], do.unflatten(0, (2, 192)))
    val, tol = packed_ref(*leaves, cu, s, do, n=16, c=8.0)
    check(got, val, tol, "packed")
    check(dict(zip(("o", "dq", "dk", "dv", "dsink"), (o, *grads))), val, tol, "flash")  # alpha = 2^-6: exact


def test_repeats_are_bit_identical_and_other_streams_agree():
    leaves, s, do, cu = _inputs([130, 257, 3], 8, 2, 128, seed=10)
    first = _run(leaves, s, do, cu, 16, 8.0)
    again = _run(leaves, s, do, cu, 16, 8.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = _run(leaves, s, do, cu, 16, 8.0)
    torch.cuda.current_stream().wait_stream(side)
    for name in first:
        assert torch.equal(first[name], again[name]) and torch.equal(first[name], third[name]), name


@pytest.mark.parametrize("H,Hkv,N", [(4, 2, 400), (16, 1, 2200)], ids=["whole", "ranges"])
def test_one_captured_graph_serves_any_lengths(H, Hkv, N):
    """Forward and backward captured once for N tokens and 5 sequences, replayed for other lengths
    and inputs (one replay with scores outside the plain form) between eager calls."""
    D, f = 64, N // 400
    leaves, s, do, _ = _inputs([N], H, Hkv, D, seed=11)
    cut = torch.tensor([0, 10, 150, 150, 290 * f, N], dtype=torch.int32, device="cuda")
    op = _op()

    def step():
        o = op(*leaves, cut, s, n=16, c=8.0)
        return [o, *torch.autograd.grad(o, [*leaves, s], do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    torch.cuda.synchronize()
    for i, (cu, scale) in enumerate([([0, 10, 150, 150, 290 * f, N], 1.0), ([0, 0, 0, N - 1, N, N], 30.0),
                                     ([0, 80, 160, 240, 320, 321], 1.0)]):
        new = _inputs([N], H, Hkv, D, scale=scale, seed=20 + i)
        with torch.no_grad():
            for dst, src in zip((*leaves, s, do), (*new[0], new[1], new[2])):
                dst.copy_(src)
            cut.copy_(torch.tensor(cu, dtype=torch.int32))
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        for rep in range(2):
            print(f"[packed] replay {i}.{rep}", flush=True)
            graph.replay()
            torch.cuda.synchronize()
            for name, a, b in zip(("o", "dq", "dk", "dv", "dsink"), static, want):
                assert torch.equal(a, b), (i, rep, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("shape", [(4,), (1, 4, 1, 1), ()])
def test_sinks_of_other_types_shapes_and_places(dtype, shape):
    """The sink's gradient comes back in its type, shape and device; one more rounding, of that type."""
    leaves, s, do, cu = _inputs([70, 33], 4, 2, 64, sink="heads" if shape else "one", seed=14)
    for dev in ("cuda", "cpu"):
        sink = s.detach().to(device=dev, dtype=dtype).reshape(shape).requires_grad_(True)
        got = _run(leaves, sink, do, cu, 16, 8.0)
        assert got["dsink"].shape == sink.shape and got["dsink"].dtype == dtype and got["dsink"].device == sink.device
        val, tol = packed_ref(*leaves, cu, sink.detach().float().cuda().reshape(-1), do, n=16, c=8.0)
        tol["dsink"] = tol["dsink"] + torch.finfo(dtype).eps / 2 * val["dsink"].abs()
        got["dsink"] = got["dsink"].cuda()
        check(got, val, tol)
    if shape:  # every other entry of a longer vector
        wide = s.detach().repeat_interleave(2)[::2].requires_grad_(True)
        got = _run(leaves, wide, do, cu, 16, 8.0)
        check(got, *packed_ref(*leaves, cu, wide, do, n=16, c=8.0))


def test_no_tokens():
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    k = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    v = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    s = torch.zeros(4, device="cuda", requires_grad=True)
    o = _op()(q, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"), s)
    grads = torch.autograd.grad(o, (q, k, v, s), torch.empty_like(o))
    assert o.shape == q.shape and [g.shape for g in grads] == [q.shape, k.shape, v.shape, s.shape] and not grads[3].any()


def test_saved_state_survives_a_hook_that_narrows_floats():
    """Saved floating tensors packed in bf16 (they are bf16 already) leave the statistic alone."""
    leaves, s, do, cu = _inputs([100], 2, 1, 64, scale=30.0, seed=12)
    narrow = torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.to(torch.bfloat16) if t.is_floating_point() and t.numel() > 8 else t, lambda t: t)
    with narrow:
        got = _run(leaves, s, do, cu, 16, 8.0)
    want = _run(leaves, s, do, cu, 16, 8.0)
    for name in got:
        assert torch.equal(got[name], want[name]), name

"""GPU: the residual stream's addition with its RMS norm, its 8-bit output and its gradients, against
float64. Bounds count roundings, u = 2^-8 of bf16 and 2^-4 of e4m3; F is the share of f32
arithmetic (sums of up to 4096 terms)."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF = torch.bfloat16
U, U8, F = 2.0 ** -8, 2.0 ** -4, 1e-5


def _ops():
    from algebraic_amd.kernels.norm import add_rms_norm, add_rms_norm_fp8
    return add_rms_norm, add_rms_norm_fp8


def _inputs(rows, d, gain, seed=0, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + rows + d)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, r, dy, ds = (scale * rn(rows, d)).to(BF), (2 * scale * rn(rows, d)).to(BF), rn(rows, d).to(BF), rn(rows, d).to(BF)
    return x, r, (1 + 0.2 * rn(d)) if gain else None, dy, ds


def _ref(s, gain, eps=1e-5):
    s = s.double()
    rms = (s.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return s / rms * (1.0 if gain is None else gain.detach().double()), rms


def _near(got, want, tol, what):
    off = ((got.double() - want).abs() / (tol + 1e-30)).max().item() if got.numel() else 0.0
    print(f"  {what}: {off:.3f} of the bound", flush=True)
    assert off <= 1.0, (what, off)


SIZES = [(1, 8), (3, 72), (5, 520), (257, 2048), (64, 4096), (1030, 768), (2, 3592), (4099, 1032)]


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("gain", [True, False])
def test_forward_and_gradients(rows, d, gain):
    x, r, g, dy, ds = _inputs(rows, d, gain)
    print(f"[add_norm] {rows}x{d} gain {gain}", flush=True)
    x.requires_grad_(True), r.requires_grad_(True)
    if gain:
        g.requires_grad_(True)
    y, s = _ops()[0](x, r, g)
    assert torch.equal(s, x.detach() + r.detach())
    want, rms = _ref(s.detach(), g)
    _near(y.detach(), want, U * want.abs() + F * want.abs(), "y")
    grads = torch.autograd.grad((y, s), [x, r] + ([g] if gain else []), (dy, ds))
    a = dy.double() * (1.0 if g is None else g.detach().double())
    h = s.detach().double()
    dh = a / rms - h * (a * h).mean(-1, keepdim=True) / rms ** 3 + ds.double()
    mag = a.abs() / rms + h.abs() * (a * h).abs().mean(-1, keepdim=True) / rms ** 3 + ds.double().abs()
    assert torch.equal(grads[0], grads[1])
    _near(grads[0], dh, U * dh.abs() + F * mag, "dx")
    if gain:
        terms = dy.double() * h / rms
        _near(grads[2], terms.sum(0), F * terms.abs().sum(0), "dgain")


def test_one_output_alone_and_a_bf16_gain():
    x, r, g, dy, ds = _inputs(33, 256, True)
    g = g.to(BF).requires_grad_(True)
    x.requires_grad_(True)
    both = torch.autograd.grad(_ops()[0](x, r, g), (x, g), (dy, torch.zeros_like(ds)))
    alone = torch.autograd.grad(_ops()[0](x, r, g)[0], (x, g), dy)
    assert torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1]) and alone[1].dtype == BF
    stream = torch.autograd.grad(_ops()[0](x, r, g)[1], x, ds)[0]
    assert torch.equal(stream, ds)
    # The norm as rms_norm computes it of the stored sum.
    from algebraic_amd.kernels.norm import rms_norm
    y, s = _ops()[0](x, r, g)
    assert torch.equal(y, rms_norm(s, g))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_gains_of_other_types_and_places(dtype):
    x, r, g, dy, ds = _inputs(20, 128, True, seed=9)
    for gain in (g.to(dtype), g.to(dtype).cpu(), g.to(dtype).repeat_interleave(2)[::2], g.to(dtype)[None]):
        gain = gain.detach().requires_grad_(True)
        y, s = _ops()[0](x, r, gain)
        want, rms = _ref(s.detach(), gain.cuda().reshape(-1))
        _near(y.detach(), want, (U + F) * want.abs(), "y")
        dg = torch.autograd.grad((y, s), gain, (dy, ds))[0]
        assert dg.shape == gain.shape and dg.dtype == dtype and dg.device == gain.device
        terms = dy.double() * s.detach().double() / rms
        _near(dg.cuda().reshape(-1), terms.sum(0), F * terms.abs().sum(0) + torch.finfo(dtype).eps / 2 * terms.sum(0).abs(), "dgain")
        y8, scale, _ = _ops()[1](x, r, gain.detach())
        _near(y8.float() * scale, want, U8 * want.abs() + (2.0 ** -10) * scale.double() + F * want.abs(), "y8")


def test_gradients_against_differences():
    """The bf16 gradient along a direction, against central differences of the float64 statement."""
    x, r, g, dy, ds = _inputs(7, 64, True, seed=5)
    x.requires_grad_(True), g.requires_grad_(True)
    y, s = _ops()[0](x, r, g)
    dx, dg = torch.autograd.grad((y, s), (x, g), (dy, ds))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    vx = torch.randn(7, 64, device="cuda", generator=gen, dtype=torch.float64)
    vg = torch.randn(64, device="cuda", generator=gen, dtype=torch.float64)
    h = 1e-6

    def f(t):
        st = s.detach().double() + t * vx  # the sum's own rounding has no derivative: around what is stored
        return (_ref(st, g.detach().double() + t * vg)[0] * dy.double()).sum() + (st * ds.double()).sum()

    slope = (f(h) - f(-h)) / (2 * h)
    terms = (dx.double() * vx).abs().sum() + (dg.double() * vg).abs().sum()
    assert abs((dx.double() * vx).sum() + (dg.double() * vg).sum() - slope) <= (U + 1e-4) * terms


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("gain", [True, False])
def test_eight_bits(rows, d, gain):
    x, r, g, _, _ = _inputs(rows, d, gain, seed=3)
    print(f"[add_norm] fp8 {rows}x{d} gain {gain}", flush=True)
    y8, scale, s = _ops()[1](x, r, g)
    assert y8.dtype == torch.float8_e4m3fn and scale.shape == (rows, 1) and torch.equal(s, x + r)
    want, _ = _ref(s, g)
    _near(scale, want.abs().amax(-1, keepdim=True) / 448, F * want.abs().amax(-1, keepdim=True) / 448, "scale")
    # Normal e4m3 values move by u8 of themselves, those under 2^-6 by half of 2^-9.
    _near(y8.float() * scale, want, U8 * want.abs() + (2.0 ** -10) * scale.double() + F * want.abs(), "y8")
    assert (y8.float().abs().amax(-1) == 448).all()


def test_eight_bits_of_special_rows():
    x = torch.zeros(6, 64, dtype=BF, device="cuda")
    r = torch.zeros_like(x)
    x[1, 5] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 1e-30
    x[4] = 1e15
    r[5], x[5] = 3.0, -3.0
    y8, scale, s = _ops()[1](x, r)
    v = y8.float() * scale
    assert not v[0].any() and not v[5].any() and (scale[[0, 5]] == 1).all()
    assert torch.isnan(v[1]).all()
    y, _ = _ops()[0](x, r)
    assert torch.equal(torch.isnan(v), torch.isnan(y.float()))
    want, _ = _ref(s[3:5], None)
    assert ((v[3:5].double() - want).abs() <= U8 * want.abs()).all()


def test_shapes_strides_streams_and_capture():
    x, r, g, dy, ds = _inputs(40, 128, True)
    y, s = _ops()[0](x.view(2, 20, 128), r.view(2, 20, 128), g)
    assert y.shape == (2, 20, 128) and s.shape == (2, 20, 128)
    wide = torch.empty(40, 200, dtype=BF, device="cuda")
    wide[:, 3:131] = x
    assert torch.equal(_ops()[0](wide[:, 3:131], r, g)[0], y.view(40, 128))
    e = torch.empty(0, 128, dtype=BF, device="cuda", requires_grad=True)
    y0, s0 = _ops()[0](e, e.detach(), g)
    assert y0.shape == (0, 128) and torch.autograd.grad((y0, s0), e, (y0, s0))[0].shape == (0, 128)
    assert _ops()[1](e.detach(), e.detach(), g)[1].shape == (0, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, _ = _ops()[0](x, r, g)
        _ops()[1](x, r, g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y2, y.view(40, 128))
    x.requires_grad_(True), g.requires_grad_(True)

    def step():
        return [*torch.autograd.grad(_ops()[0](x, r, g), (x, g), (dy, ds)), *_ops()[1](x.detach(), r, g.detach())]

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(40, 128, device="cuda"))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i

"""GPU: the operators between one token and the next at the edges of what they take."""

import math

import pytest

from test_step_gpu import BF, F32, F64, _check_sample, _gen, _sample

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

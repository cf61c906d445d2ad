"""CPU: what the packed, paged and residual-norm entry points make of calls at the edges of what they
take, before anything is launched."""

import pytest

torch = pytest.importorskip("torch")

BF = torch.bfloat16


@pytest.mark.parametrize("heads,D", [(4, 64), (1, 128), (3, 64)])
@pytest.mark.parametrize("ts", [0, 1, 4, 60, 260, 1 << 28, 1 << 33])
def test_one_token_has_any_token_stride(heads, D, ts):
    """torch calls one token's rows contiguous whatever its stride: what the kernels are given holds."""
    from algebraic_amd.kernels.packed import _rows
    t = torch.randn(1, heads, D).to(BF)
    for hs in (D, 1) if heads == 1 else (D,):
        view = torch.as_strided(t, t.shape, (ts, hs, 1))
        got, (at, got_ts, got_hs) = _rows(view)
        assert at == got.data_ptr() == t.data_ptr() and torch.equal(got, t)  # read in place
        assert got_ts >= D and got_hs >= D and not (got_ts | got_hs) % 8 and 66 * got_ts + heads * got_hs + D < 1 << 30


def test_rows_that_are_copied_and_rows_that_are_read_in_place():
    from algebraic_amd.kernels.packed import _rows
    base = torch.randn(5, 3, 128).to(BF)
    for t, copied in ((base, False), (base[..., :64], False), (base.transpose(0, 1), False), (base[..., 1:65], True),
                      (base[:, :1].expand(-1, 3, -1), True), (base[:1].expand(5, -1, -1), True),
                      (base[:1, :1].expand(1, 3, -1), True), (base[:1, :, 1:65], True), (base.reshape(5, 128, 3).transpose(1, 2), True)):
        got, (at, ts, hs) = _rows(t)
        D = t.shape[2]
        assert (at != t.data_ptr()) == copied and torch.equal(got, t)
        assert ts >= D and hs >= D and not (ts | hs) % 8 and at == got.data_ptr()
        again = torch.as_strided(got, t.shape, (ts, hs, 1))
        assert torch.equal(again, t)


def test_one_page_and_one_head_have_any_stride():
    from algebraic_amd.kernels.paged import _pages
    t = torch.zeros(1, 1, 16, 64, dtype=BF)
    for ps, hs in ((1, 1), (0, 0), (12, 20), (1 << 35, 1 << 34)):
        at, *strides = _pages("k_pages", torch.as_strided(t, t.shape, (ps, hs, 64, 1)), 1, 64, t.device)
        assert at == t.data_ptr() and all(x >= 64 and x % 8 == 0 for x in strides) and strides[2] == 64
    with pytest.raises(ValueError, match="contiguous"):
        _pages("k_pages", torch.as_strided(t, t.shape, (1024, 1024, 60, 1)), 1, 64, t.device)

"""CPU: what the packed, paged and residual-norm entry points make of calls at the edges of what they
take, before anything is launched."""

import ctypes

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


def test_sizes_past_one_launch_are_refused():
    """A launch has fewer than 2^32 threads: said before anything runs, and no count wraps at 2^32."""
    from algebraic_amd import _lib
    from algebraic_amd.kernels.norm import add_rms_norm, add_rms_norm_fp8
    h, P = _lib.load(), ctypes.c_void_p(16)

    def unsupported(rc, text):
        assert rc == _lib.ALG_ERR_UNSUPPORTED and text.encode() in h.alg_last_error(), (rc, h.alg_last_error())

    def append(N):
        return h.alg_paged_append(None, N, 1, 1, 1, 64, P, 64, 64, P, 64, 64, P, 64, 64, P, 1024, 1024, 64, P, 1024, 1024, 64,
                                  4, 16, P, 2, P, P, None, None, 1, None, None, 0, 1e-5, P)

    for N in (1 << 24, 1 << 27):
        unsupported(append(N), "tokens")
    for rows in ((1 << 26) - 3, 1 << 26, (1 << 31) - 1):
        unsupported(h.alg_add_rms_norm_fwd(None, rows, 64, P, P, None, 1, 1e-5, P, P, P), "rows")
        unsupported(h.alg_add_rms_norm_fp8(None, rows, 64, P, P, None, 1, 1e-5, P, P, P), "rows")
    for rows in (1 << 26, (1 << 32) + 5):
        x = torch.empty(rows, 8, dtype=BF, device="meta")
        for op in (add_rms_norm, add_rms_norm_fp8):
            with pytest.raises(NotImplementedError, match="rows"):
                op(x, x)

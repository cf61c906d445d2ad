"""CPU: what the operators between one token and the next make of calls at the edges of what they take, before
anything is launched."""

import math

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("top_k", [0.5, 2.9, math.inf])
def test_a_top_k_that_is_no_whole_number(top_k):
    """A number as a tensor: whole or refused (0.5 would else be 0, which cuts nothing)."""
    from algebraic_amd import head_sample
    z, u = torch.zeros(3, 50), torch.zeros(3)
    with pytest.raises(ValueError, match="top_k must hold whole numbers"):
        head_sample(z, u, top_k=top_k)


@pytest.mark.parametrize("top_k", [0, 7, 7.0, 1 << 40, 1 << 2000, True])
def test_a_whole_top_k(top_k):
    from algebraic_amd import head_sample
    with pytest.raises(RuntimeError, match="GPU"):  # the last of the checks
        head_sample(torch.zeros(3, 50), torch.zeros(3), top_k=top_k)

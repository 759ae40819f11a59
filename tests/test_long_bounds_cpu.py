"""Bounds on the context length up to the largest whole number of their type."""
import pytest

from vasr_paged_attn import _lib

MOST = 2 ** 31 - 1


@pytest.mark.parametrize("d,bs", [(64, 8), (64, 32), (128, 8), (128, 16), (128, 32), (256, 16)])
@pytest.mark.parametrize("seqs,window,rows,heads", [(1, 1, 1, 16), (64, 5, 1, 16), (1, 8, 8, 8)])
def test_scored_workspace_of_long_bounds(d, bs, seqs, window, rows, heads):
    """The raw scores alone need 4 bytes a scored row and token, and the size follows the bound."""
    size = _lib.lib().vasr_pa_paged_attention_scored_workspace_size
    last = 0
    for bound in (2 ** 20, 2 ** 30, MOST - 4096, MOST - 1200, MOST - 40, MOST - 1, MOST):
        need = size(seqs, window, rows, heads, 8, d, bs, bound)
        assert need >= seqs * rows * heads * 4 * bound
        assert need < 2 ** 50 and need >= last
        last = need

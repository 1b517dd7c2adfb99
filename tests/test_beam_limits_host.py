"""How many continuations a selection may be asked for, without a GPU."""
import pytest

from kvmix_b200 import beams, paged
from test_beam_host import select


@pytest.mark.parametrize("b,ends,V,want", [(1, 0, 100, 2), (4, 0, 100, 8), (4, 1, 100, 8), (4, 2, 100, 12), (64, 0, 100, 128), (64, 1, 100, 128), (4, 31, 1000, 128), (1, 127, 1000, 128),
                                           (2, 50, 3, 6), (1, 0, 1, 1), (64, 5, 1, 64)])
def test_as_many_as_leave_the_beams(b, ends, V, want):
    assert beams._how_many(None, b, ends, V) == want


@pytest.mark.parametrize("b,ends,V", [(64, 2, 1000), (4, 32, 1000), (1, 128, 1000), (3, 42, 50)])
@pytest.mark.parametrize("n", [None, 128])
def test_more_ends_than_can_be_told_apart(b, ends, V, n):
    """The refusal names what is too many, not a range that is empty."""
    with pytest.raises(RuntimeError, match=r"beams \* \(1 \+ number of ends\) is at most 128"):
        beams._how_many(n, b, ends, V)


@pytest.mark.parametrize("n,b,ends,V,low,high", [(7, 4, 1, 100, 8, 128), (129, 4, 1, 100, 8, 128), (0, 1, 0, 5, 1, 5), (7, 3, 9, 2, 6, 6)])
def test_out_of_range(n, b, ends, V, low, high):
    with pytest.raises(RuntimeError, match=f"n must be {low} to {high} "):
        beams._how_many(n, b, ends, V)


@pytest.mark.parametrize("V", [1 << 24, (1 << 31) - 4096, (1 << 31) - 4095, (1 << 31) - 1])
def test_parts_of_the_widest_rows(V):
    """One row is 32 parts however wide it is."""
    n = 8
    assert paged._library().kvq_beam_select_workspace_bytes(select(requests=1, beams=1, vocabulary=V, n=n)) == 32 * (8 * n + 16)

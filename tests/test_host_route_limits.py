"""The router's largest rows: the kernel steps through a row by 256 columns in 32 bits, which has to end before 2^31."""
import pytest

A = 1 << 20          # an aligned address; every call below is refused before anything reads it
SHAPE = -1


@pytest.mark.parametrize("K", [0x7ffffff0, 0x7fffff08, 1 << 31, 1 << 40])
def test_rows_whose_last_step_would_overflow_are_refused(pkg, K):
    assert pkg._lib.load().gmlp_moe_route(4, K, 8, 2, 1, 0, A, K, A, A, A, None) == SHAPE

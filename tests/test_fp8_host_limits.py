"""Sizes beyond what rows' sums count with are refused before anything is launched (no GPU needed)."""
import pytest

SOME = 1 << 20                                                    # aligned, never followed


@pytest.mark.parametrize("top", [1 << 31, (1 << 32) - 32, (1 << 32) - 1])
def test_sums_over_more_places_than_are_counted_are_refused(spg, top):
    """A count that goes up to 32 places beyond top_k would begin again at zero."""
    lib = spg.lib()
    assert lib.spgk_combine_rows(SOME, 2, 10, 8, SOME, SOME, 1, top, 10, SOME, 2, 10, None) == -2
    assert b"spgk_combine_rows" in lib.spgk_error_string()

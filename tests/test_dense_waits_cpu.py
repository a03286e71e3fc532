"""Settings of the int8 products' bounded waits: their bounds, without a GPU."""

import pytest

import megamoe
from megamoe import _lib


def test_wait_budget_bounds():
    for bad in (0, -5, 60_000_001):
        with pytest.raises(ValueError):
            megamoe.int8_set_wait_budget(bad)
    for good in (1, 60_000_000, 1_500_000):
        megamoe.int8_set_wait_budget(good)
    L = _lib.lib()
    for rank, launches in ((-1, 1), (8, 1), (0, -1)):
        assert L.mm_int8_withhold(rank, launches) == _lib.MM_ERR_INVALID

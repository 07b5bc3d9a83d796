"""Limits of the grouped products' barrier waits that are refused."""
import pytest


@pytest.mark.parametrize("seconds", [-1.0, -1e-9, 61.0])
def test_refused_limits(seconds):
    from dsmezo_b200 import DsmzError, grouped
    with pytest.raises(DsmzError, match="0 to 60 s"):
        grouped.set_wait_limit(seconds)


def test_limits_are_accepted_and_restored():
    from dsmezo_b200 import grouped
    for s in (0.0, 1e-9, 60.0, 1.0):
        grouped.set_wait_limit(s)

"""What the cache operators decide on the host, against brute force."""
import itertools

import pytest

from rapid_h3_b200 import kv_cache


@pytest.mark.parametrize("t,heads", [(1, 1), (1, 4), (5, 1), (2, 2), (3, 4), (4, 3), (7, 5)])
def test_overlapping_rows_are_found(t, heads):
    d, found = 8, set()
    for st, sh in itertools.product(range(0, 80, 2), repeat=2):
        at = sorted(i * st + h * sh for i in range(t) for h in range(heads))
        overlap = any(b - a < d for a, b in zip(at, at[1:]))
        assert kv_cache._rows_overlap(t, heads, d, st, sh) == overlap, (st, sh)
        found.add(overlap)
    assert found == ({False} if t == heads == 1 else {False, True})

"""The counts of visible keys that the timed cases' operations are reckoned from (perf/operators.py)."""
import random

import pytest

from perf import operators as ops


@pytest.mark.parametrize("causal,window,sinks", [(False, 0, 0), (True, 0, 0), (True, 1, 0), (True, 1, 3), (True, 7, 0), (True, 7, 2), (True, 7, 40), (True, 64, 5)])
def test_sum_of_visible_keys(causal, window, sinks):
    c = {"causal": causal, "window": window, "sinks": sinks}
    rng = random.Random(window + sinks)
    for p0, q in [(0, 1), (0, 7), (0, 8), (3, 5), (6, 1), (7, 1), (200, 1), *((rng.randint(0, 90), rng.randint(1, 90)) for _ in range(60))]:
        n = p0 + q
        seen = [n if not causal else sum(j <= p and (not window or p - j < window or j < sinks) for j in range(n)) for p in range(p0, n)]
        assert [ops._visible(p, n, c) for p in range(p0, n)] == seen
        assert ops._visible_sum(p0, q, n, c) == sum(seen)

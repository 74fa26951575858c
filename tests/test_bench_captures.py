"""bench.without_captures: means over the steps that captured no graph."""
import pytest

import bench


def step(ms, tokens, captured=0):
    return {"ms": ms, "tokens": tokens, "captured": captured}


def test_steps_that_captured_are_left_out():
    mean, n = bench.without_captures([step(8.0, 90), step(21.0, 40, 1), step(9.0, 60), step(34.0, 50, 2)])
    assert n == 2 and mean["ms"] == 8.5 and mean["tokens"] == 75


def test_all_count_without_captures():
    mean, n = bench.without_captures([step(8.0, 90), step(10.0, 60)])
    assert (mean["ms"], mean["tokens"], n) == (9.0, 75.0, 0)


def test_all_count_where_each_one_captured():
    mean, n = bench.without_captures([step(20.0, 90, 1), step(30.0, 60, 1)])
    assert (mean["ms"], n) == (25.0, 2)


@pytest.mark.parametrize("steps", [1, 7])
def test_the_mean_is_the_total_over_the_steps(steps):
    mean, _ = bench.without_captures([step(float(i), 10 * i) for i in range(steps)])
    assert mean["ms"] * steps == pytest.approx(sum(range(steps)))

"""A thread that fails or hangs is seen by the tests that start it."""

import threading

import pytest
from side_by_side import run_threads


def test_all_passes_are_made():
    counts = [0, 0, 0]

    def work(i):
        counts[i] += 1

    run_threads([lambda i=i: work(i) for i in range(3)], 5)
    assert counts == [5, 5, 5]


@pytest.mark.parametrize("at", [0, 4])
def test_what_a_thread_raises_is_raised(at):
    seen = []

    def fail():
        seen.append(None)
        if len(seen) > at:
            raise RuntimeError("planted")

    with pytest.raises(RuntimeError, match="planted"):
        run_threads([lambda: None, fail], 5)


def test_a_thread_that_waits_is_named():
    never = threading.Event()
    with pytest.raises(AssertionError, match="passes made"):
        run_threads([lambda: None, lambda: never.wait(30)], 2, timeout=0.2)
    never.set()

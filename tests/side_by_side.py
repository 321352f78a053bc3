"""Passes of several threads at once, for the tests."""

import threading


def run_threads(works, passes, timeout=60.0):
    """Calls each of ``works`` ``passes`` times, in a thread of its own.
    Raises the first thing that one of them raised, and AssertionError where
    one has not made all of its passes in time."""
    raised, made = [], [0] * len(works)

    def run(i):
        try:
            for _ in range(passes):
                works[i]()
                made[i] += 1
        except BaseException as error:  # a thread's end is silent otherwise
            raised.append(error)

    threads = [threading.Thread(target=run, args=(i,), daemon=True) for i in range(len(works))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout)
    if raised:
        raise raised[0]
    assert made == [passes] * len(works), f"passes made: {made} of {passes}"

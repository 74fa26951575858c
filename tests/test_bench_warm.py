"""bench.timed_warm: the run that counts captured no graphs, and each run starts from the same state."""
from types import SimpleNamespace

import bench


def engine(shapes_per_run):
    """An engine whose i-th run meets the given shapes and appends one token per shape."""
    seqs = [SimpleNamespace(tokens=[1, 2, 3], outputs=[3], num_computed=2) for _ in range(2)]
    eng = SimpleNamespace(graphs={}, sched=SimpleNamespace(running=seqs), starts=[], i=0)

    def timed():
        eng.starts.append([(list(s.tokens), list(s.outputs), s.num_computed) for s in seqs])
        for shape in shapes_per_run[eng.i]:
            eng.graphs.setdefault(shape, object())
            for s in seqs:
                s.tokens.append(9)
                s.outputs.append(9)
                s.num_computed += 1
        eng.i += 1
        return eng.i
    return eng, timed


def test_a_run_without_captures_counts_at_once():
    eng, timed = engine([[]])
    assert bench.timed_warm(eng, timed) == (1, 0)


def test_a_run_that_captures_is_repeated_from_the_same_sequences():
    eng, timed = engine([[1, 2, 3], [1, 2, 3]])
    assert bench.timed_warm(eng, timed) == (2, 0)
    assert eng.starts[0] == eng.starts[1] and len(eng.sched.running[0].tokens) == 6


def test_the_last_run_counts_and_says_what_it_captured():
    eng, timed = engine([[1], [2], [3]])
    assert bench.timed_warm(eng, timed) == (3, 1)
    assert eng.starts[0] == eng.starts[1] == eng.starts[2]


def test_ranks_repeat_together():
    eng, timed = engine([[], []])
    others = iter([2, 0])  # another rank captured two
    assert bench.timed_warm(eng, timed, lambda n: max(n, next(others))) == (2, 0)

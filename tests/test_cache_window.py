"""CPU: the books of evicted pages and of steps planned ahead."""
import random

import pytest
import torch

from qlinear import cache as C
from test_cache import small, write  # noqa: F401


def seen(n, window, sinks):
    """What some token at position n or later sees."""
    return [j for j in range(n) if j > n - window or j < sinks]


@pytest.mark.parametrize("seed", range(8))
def test_what_the_window_sees_stays(small, seed):  # noqa: F811
    rng = random.Random(seed)
    window, sinks = rng.choice([(1, 0), (16, 4), (20, 16), (33, 17), (100, 1)])
    c, want, count = small(60), {}, 0
    for _ in range(200):
        op = rng.choice(["new", "step", "step", "step", "fork", "free", "evict", "evict", "compact"])
        if op == "new" or not want:
            want[c.new()] = []
        elif op == "step":
            q, n = rng.choice(sorted(want)), rng.choice([1, 1, 5, 16, 40])
            try:
                s = c.step([q], [n])
            except C.OutOfPages:
                victim = max(want, key=lambda x: len(want[x]))
                c.free(victim)
                del want[victim]
                continue
            values = [float(count + i) for i in range(n)]
            count += n
            write(c, s, values)
            want[q] += values
        elif op == "fork":
            q = rng.choice(sorted(want))
            want[c.fork(q)] = list(want[q])
        elif op == "free":
            q = rng.choice(sorted(want))
            c.free(q)
            del want[q]
        elif op == "evict":
            q = rng.choice(sorted(want))
            free, gone = c.free_pages, c.evict(q, window, sinks)
            assert c.free_pages <= free + gone
            kept = {j // c.page_size for j in seen(len(want[q]), window, sinks)}
            for i, p in enumerate(c.pages_of(q)):
                # what is seen is there; a page that neither holds anything seen nor may be written is not
                assert p >= 0 if i in kept or (i + 1) * c.page_size > len(want[q]) else p == -1
            if gone:
                with pytest.raises(ValueError):
                    c.truncate(q, len(want[q]) - 1)
                c.truncate(q, len(want[q]))
        else:
            c.compact()
            used = {p for q in want for p in c.pages_of(q)} - {-1}
            assert used == set(range(len(used)))
        for q, v in want.items():
            for j in seen(len(v), window, sinks):
                page = c.pages_of(q)[j // c.page_size]
                assert page >= 0 and float(c.pool[1, 0, page, 0, j % c.page_size, 1]) == v[j]
        assert c.free_pages == c.pages - len({p for q in want for p in c.pages_of(q)} - {-1})


def test_evict_refusals(small):  # noqa: F811
    c = small(4)
    a = c.new()
    for bad in ((0, 0), (-1, 0), (4, -1)):
        with pytest.raises(ValueError):
            c.evict(a, *bad)
    assert c.evict(a, 5, 1) == 0  # nothing there
    with pytest.raises(KeyError):
        c.evict(99, 5)


@pytest.mark.parametrize("done", [0, 1, 17, 40])
def test_ahead_enters_the_steps_that_ran(small, done):  # noqa: F811
    """The same pages in the same order as single steps; the others go back."""
    c, d = small(20), small(20)
    for x in (c, d):
        seqs = [x.new() for _ in range(3)]
        x.step(seqs, [1, 16, 30])
        seqs.append(x.fork(seqs[2]))  # shares a partly filled page
    a = c.ahead(seqs, 40)
    assert c.free_pages == 20 - 6 - 8 - 2 and a.max_kv == 70
    for refused in (lambda: c.step([seqs[0]], [1]), lambda: c.fork(seqs[1]), lambda: c.free(seqs[2]), lambda: c.truncate(seqs[0], 0), c.compact,
                    lambda: c.evict(seqs[3], 4), lambda: c.ahead([seqs[3]], 1)):
        with pytest.raises(ValueError):
            refused()
    other = c.new()
    c.step([other], [3])  # the rest of the cache goes on
    c.free(other)
    with pytest.raises(ValueError):
        a.close(41)
    a.close(done)
    a.close(done)  # once is enough
    for _ in range(done):
        d.step(seqs, [1] * 4)
    assert [c.length(s) for s in seqs] == [d.length(s) for s in seqs]
    assert [len(c.pages_of(s)) for s in seqs] == [len(d.pages_of(s)) for s in seqs]
    held = {p for s in seqs for p in c.pages_of(s)}
    assert c.free_pages == 20 - len(held)
    if done:
        assert d.free_pages == c.free_pages
    c.step(seqs, [1] * 4)


def test_ahead_refusals(small):  # noqa: F811
    c = small(3)
    a = c.new()
    for seqs, n in (([a], 0), ([], 3), ([a, a], 1)):
        with pytest.raises(ValueError):
            c.ahead(seqs, n)
    with pytest.raises(C.OutOfPages):
        c.ahead([a], 49)
    assert c.free_pages == 3
    c.ahead([a], 48).close(0)
    assert c.free_pages == 3 and c.length(a) == 0

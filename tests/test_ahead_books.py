"""CPU: an Ahead that a program drops can be closed all the same, and one that cannot be made leaves the cache's books as they were."""
import gc

import pytest

from qlinear import cache as C
from test_cache import small  # noqa: F401


def books(c):
    return c.free_pages, {s: (c.length(s), c.pages_of(s)) for s in c._lists}, list(c._refs)


def test_dropped_without_close(small):  # noqa: F811
    c = small(20)
    seqs = [c.new() for _ in range(3)]
    c.step(seqs, [1, 16, 30])
    before = books(c)
    idle = c.new()
    c.ahead(seqs, 40)
    gc.collect()
    # its pages are not given back by themselves: a captured step may still write them
    assert c.free_pages == before[0] - 2 - 3 - 3  # 41, 56 and 70 positions of pages of 16, less the 1, 1 and 2 pages there
    assert c.ahead_of(idle) is None and c.ahead_of(seqs[0]) is c.ahead_of(seqs[2])
    with pytest.raises(ValueError):
        c.free(seqs[0])
    c.free(idle)
    c.ahead_of(seqs[1]).close(0)
    assert books(c) == before and all(c.ahead_of(s) is None for s in seqs)
    c.step(seqs, [1] * 3)  # they are the cache's again
    c.free(seqs[0])
    c.ahead(seqs[1:], 40)
    c.ahead_of(seqs[1]).close(3)
    assert c.length(seqs[1]) == 20 and c.ahead_of(seqs[1]) is None


@pytest.mark.parametrize("what", ["zeros", "tensor"])
def test_no_memory_for_its_tensors(small, monkeypatch, what):  # noqa: F811
    c = small(20)
    seqs = [c.new() for _ in range(3)]
    c.step(seqs, [1, 16, 30])
    before = books(c)

    def fail(*a, **kw):
        raise MemoryError

    with monkeypatch.context() as m:
        m.setattr(C.torch, what, fail)
        with pytest.raises(MemoryError):
            c.ahead(seqs, 40)
    gc.collect()
    assert books(c) == before
    c.ahead(seqs, 40).close(1)
    assert [c.length(s) for s in seqs] == [2, 17, 31]


def test_refused(small):  # noqa: F811
    c = small(3)
    a = c.new()
    for n in (0, 49):
        with pytest.raises((ValueError, C.OutOfPages)):
            c.ahead([a], n)
    gc.collect()
    assert c.free_pages == 3 and c.length(a) == 0

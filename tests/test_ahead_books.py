"""CPU: an Ahead that is dropped, or that cannot be made, leaves the cache's books as they were."""
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
    ahead = c.ahead(seqs, 40)
    assert c.free_pages < before[0]
    del ahead
    gc.collect()
    assert books(c) == before
    c.step(seqs, [1] * 3)  # they are the cache's again
    c.free(seqs[0])
    # one that was closed counts as it was closed
    ahead = c.ahead(seqs[1:], 40)
    ahead.close(3)
    after = books(c)
    del ahead
    gc.collect()
    assert books(c) == after and c.length(seqs[1]) == 20


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

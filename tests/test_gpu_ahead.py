"""GPU: steps planned ahead end where their pages do, whoever asks for more of them."""
import pytest
import torch

import qlinear
from qlinear import _lib
from qlinear.cache import PagedCache

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("max_kv,room", [(70, True), (69, False), (0, False), (2 ** 31 - 1, True)])
def test_a_step_past_its_bound_has_no_room(max_kv, room):
    """Pages, columns and rows suffice; the longest sequence would hold 70."""
    table = i32([[3, 4, 5, 6, 7], [8, 9, 10, 11, 12]])
    got = qlinear.plan_step(table, i32([5, 30]), i32([1, 40]), page_size=16, max_tokens=41, max_kv=max_kv)
    if room:
        assert got[3].tolist() == [6, 70] and got[2].tolist() == [0, 1, 41] and qlinear.device_error() == 0
    else:
        assert qlinear.device_error() == _lib.DEV_ERR_NO_ROOM
        assert got[3].tolist() == [5, 30] and got[2].tolist() == [0, 0, 0] and set(got[1].tolist()) == {-1}
    for bad in (-1, 1 << 31):
        with pytest.raises(ValueError):
            qlinear.plan_step(table, i32([5, 30]), i32([1, 40]), page_size=16, max_tokens=41, max_kv=bad)


def state(ahead, step):
    return [t.tolist() for t in (step.kv_lens, step.page_table, ahead._out[4])]


@pytest.mark.parametrize("lengths", [[3, 16], [16, 32], [5]])
@pytest.mark.parametrize("steps", [1, 16, 20])
def test_replays_past_the_reserved_steps_have_no_room(lengths, steps):
    """Inside the last page and at its end."""
    cache = PagedCache(1, 1, 16, 40, 16)
    seqs = [cache.new() for _ in lengths]
    cache.step(seqs, lengths)
    ahead = cache.ahead(seqs, steps)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = ahead.next()
    for i in range(steps):
        graph.replay()
        assert step.kv_lens.tolist() == [n + i + 1 for n in lengths] and min(step.slots.tolist()) >= 0
    assert qlinear.device_error() == 0
    before = state(ahead, step)
    for _ in range(3):
        graph.replay()
        assert qlinear.device_error() == _lib.DEV_ERR_NO_ROOM
        assert set(step.slots.tolist()) == {-1} and set(step.q_starts.tolist()) == {0} and state(ahead, step) == before
    ahead.close(steps)
    assert [cache.length(s) for s in seqs] == [n + steps for n in lengths]


@pytest.mark.parametrize("done", [0, 1, 5])
def test_calls_past_the_steps_and_after_close(done):
    cache = PagedCache(1, 1, 16, 8, 16)
    seqs = [cache.new(), cache.new()]
    cache.step(seqs, [16, 15])
    ahead = cache.ahead(seqs, 5)
    for _ in range(5):
        step = ahead.next()
    with pytest.raises(ValueError):
        ahead.next()
    assert step.kv_lens.tolist() == [21, 20] and qlinear.device_error() == 0
    ahead.close(done)
    other = cache.new()  # takes what the closed one has given back
    cache.step([other], [16 * cache.free_pages])
    lent = [set(cache.pages_of(s)) for s in (*seqs, other)]
    assert sum(map(len, lent)) == len(set.union(*lent)) == 8
    before = state(ahead, step)
    for _ in range(2):
        after = ahead.next()
        assert qlinear.device_error() == _lib.DEV_ERR_NO_ROOM
        assert after.slots.tolist() == [-1, -1] and after.positions.tolist() == [0, 0] and after.q_starts.tolist() == [0, 0, 0]
        assert state(ahead, step) == before
    assert qlinear.device_error() == 0

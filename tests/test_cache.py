"""CPU: the paged cache's books (page lists, sharing, copy on write, compaction), with the copy of
pages replaced by the same copy in torch; random histories against plain lists of tokens."""
import random

import pytest
import torch

from qlinear import cache as C


@pytest.fixture
def small(monkeypatch):
    def copy(pool, src, dst):
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)  # what copy_pages asks for
        pool[:, :, dst] = pool[:, :, src]

    monkeypatch.setattr(C.decoder, "copy_pages", copy)
    return lambda pages, ps=16: C.PagedCache(2, 1, 2, pages, ps, dtype=torch.float32, device="cpu")


def write(cache, step, values):
    """The append of a pass: value v of each new token in every layer, keys and values."""
    for slot, v in zip(step.slots.tolist(), values):
        cache.pool[:, :, slot // cache.page_size, :, slot % cache.page_size] = v


def read(cache, seq):
    pages, n = cache.pages_of(seq), cache.length(seq)
    assert len(pages) == -(-n // cache.page_size)
    return [float(cache.pool[1, 0, pages[i // cache.page_size], 0, i % cache.page_size, 1]) for i in range(n)]


def test_step_tensors(small):
    c = small(10)
    a, b = c.new(), c.new()
    s = c.step([a, b], [17, 3])
    assert s.positions.tolist() == list(range(17)) + [0, 1, 2] and s.max_q == 17 and s.max_kv == 17
    assert s.q_starts.tolist() == [0, 17, 20] and s.kv_lens.tolist() == [17, 3]
    assert s.page_table.tolist() == [c.pages_of(a), c.pages_of(b) + [-1]]
    assert s.slots.tolist() == [c.pages_of(a)[i // 16] * 16 + i % 16 for i in range(17)] + [c.pages_of(b)[0] * 16 + i for i in range(3)]
    assert s.page_table.dtype == s.q_starts.dtype == s.kv_lens.dtype == torch.int32 and s.slots.dtype == torch.int64
    s = c.step([b, a], [0, 1])
    assert s.positions.tolist() == [17] and s.q_starts.tolist() == [0, 0, 1] and s.kv_lens.tolist() == [3, 18]


@pytest.mark.parametrize("seed", range(12))
def test_random_histories(small, seed):
    rng = random.Random(seed)
    c, want, count = small(40), {}, 0
    for _ in range(300):
        op = rng.choice(["new", "step", "step", "step", "fork", "free", "truncate", "compact"])
        if op == "new" or not want:
            want[c.new()] = []
        elif op == "step":
            seqs = rng.sample(sorted(want), rng.randint(1, min(4, len(want))))
            n = [rng.choice([0, 1, 1, 5, 16, 33]) for _ in seqs]
            if not sum(n):
                continue
            before = ({s: c.pages_of(s) for s in want}, c.free_pages)
            try:
                s = c.step(seqs, n)
            except C.OutOfPages:
                assert before == ({s: c.pages_of(s) for s in want}, c.free_pages)
                victim = max(want, key=lambda x: len(want[x]))
                c.free(victim)
                del want[victim]
                continue
            values = [float(count + i) for i in range(sum(n))]
            count += sum(n)
            write(c, s, values)
            at = 0
            for q, k in zip(seqs, n):
                want[q] += values[at:at + k]
                at += k
        elif op == "fork":
            q = rng.choice(sorted(want))
            want[c.fork(q)] = list(want[q])
        elif op == "free":
            q = rng.choice(sorted(want))
            c.free(q)
            del want[q]
        elif op == "truncate":
            q = rng.choice(sorted(want))
            n = rng.randint(0, len(want[q]))
            c.truncate(q, n)
            want[q] = want[q][:n]
        else:
            c.compact()
            used = {p for q in want for p in c.pages_of(q)}
            assert used == set(range(len(used)))
        for q, v in want.items():
            assert read(c, q) == v
        assert c.free_pages == c.pages - len({p for q in want for p in c.pages_of(q)})


def test_forks_share_until_written(small):
    c = small(8)
    a = c.new()
    write(c, c.step([a], [20]), range(20))
    b, d = c.fork(a), c.fork(a)
    assert c.free_pages == 6 and c.pages_of(a) == c.pages_of(b) == c.pages_of(d)
    write(c, c.step([a, b, d], [1, 1, 1]), [100, 101, 102])  # two copy the last page, the third keeps it
    assert c.free_pages == 4 and len({c.pages_of(x)[1] for x in (a, b, d)}) == 3 and len({c.pages_of(x)[0] for x in (a, b, d)}) == 1
    assert [read(c, x)[-1] for x in (a, b, d)] == [100.0, 101.0, 102.0]


def test_refusals(small):
    c = small(2)
    a = c.new()
    for seqs, n in (([a], [1, 2]), ([a, a], [1, 1]), ([], []), ([a], [-1]), ([a], [0])):
        with pytest.raises(ValueError):
            c.step(seqs, n)
    with pytest.raises(C.OutOfPages):
        c.step([a], [33])
    assert c.free_pages == 2 and c.length(a) == 0
    with pytest.raises(ValueError):
        c.truncate(a, 1)
    with pytest.raises(KeyError):
        c.free(99)
    for bad in (dict(pages=0), dict(page_size=8), dict(page_size=24), dict(layers=0)):
        with pytest.raises(ValueError):
            C.PagedCache(**{**dict(layers=1, kv_heads=1, head_dim=2, pages=2, device="cpu"), **bad})

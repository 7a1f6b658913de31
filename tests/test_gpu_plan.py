"""GPU: the step's index tensors against lists (whole numbers: equal)."""
import random

import pytest
import torch

import qlinear
from qlinear import _lib

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(v, **I32)


def lists(table, have, new, ps, rows, free=None, taken=0):
    table = [list(r) for r in table]
    positions, slots, starts = [], [], [0]
    for b, (h, n) in enumerate(zip(have, new)):
        for at in range(h, h + n):
            if free is not None and at % ps == 0:
                table[b][at // ps] = free[taken]
                taken += 1
            positions.append(at)
            slots.append(table[b][at // ps] * ps + at % ps)
        starts.append(len(positions))
    pad = rows - len(positions)
    return (positions + [0] * pad, slots + [-1] * pad, starts, [h + n for h, n in zip(have, new)], taken), table


def check(have, new, ps, extra_rows=0, extra_columns=0, grow=True, taken=0, seed=0):
    rng = random.Random(seed)
    B, rows = len(have), sum(new) + extra_rows
    need = [-(-(h + n) // ps) for h, n in zip(have, new)]
    held = [-(-h // ps) for h in have] if grow else need
    width = max(need + [0]) + extra_columns
    pages = rng.sample(range(1 << 20), sum(need) + taken)
    table, at = [], 0
    for n in held:
        table.append(pages[at:at + n] + [-7] * (width - n))
        at += n
    free = pages[at:] if grow else None
    want, after = lists(table, have, new, ps, rows, free, taken)
    t = i32(table).view(B, width)
    got = qlinear.plan_step(t, i32(have).view(B), i32(new).view(B), page_size=ps, max_tokens=rows,
                            free_pages=i32(free) if grow else None, taken=i32([taken]) if grow else None)
    for g, w, d in zip(got, want, (torch.int64, torch.int64, torch.int32, torch.int32)):
        assert g.dtype == d and g.tolist() == w
    assert (got[4].tolist() == [want[4]]) if grow else got[4] is None
    assert t.tolist() == after
    assert qlinear.device_error() == 0


@pytest.mark.parametrize("grow", [True, False])
@pytest.mark.parametrize("ps", [1, 16, 64, 1024])
@pytest.mark.parametrize("have,new", [
    ([0], [1]), ([15], [1]), ([16], [1]), ([17], [0]), ([0], [0]), ([0, 0, 5], [0, 3, 0]), ([0], [4097]), ([31, 0, 700], [1, 1000, 33]),
    ([1023] * 40, [1] * 40), ([5000, 0], [1, 9000]), ([0] * 33, list(range(33)))])
def test_plans(have, new, ps, grow):
    check(have, new, ps, grow=grow)
    check(have, new, ps, extra_rows=77, extra_columns=5, grow=grow, taken=3 * grow, seed=1)


@pytest.mark.parametrize("seed", range(8))
def test_random_plans(seed):
    rng = random.Random(seed)
    B = rng.choice([1, 3, 64, 1000, 1025, 4000, 9000])
    most = max(1, 20000 // B)
    have = [rng.choice([0, rng.randrange(200), 16 * rng.randrange(20)]) for _ in range(B)]
    new = [rng.choice([0, 1, 1, rng.randrange(most + 1)]) for _ in range(B)]
    check(have, new, rng.choice([16, 32]), extra_rows=rng.randrange(3000), grow=bool(seed % 3), taken=rng.randrange(9) * bool(seed % 3), seed=seed)


def test_no_sequences_and_no_rows():
    check([], [], 16, extra_rows=5)
    check([], [], 16, grow=False)
    check([3, 4], [0, 0], 16, extra_rows=0)
    # an empty list of free pages, where none is needed
    got = qlinear.plan_step(i32([[4]]), i32([3]), i32([2]), page_size=16, max_tokens=2, free_pages=i32([]), taken=i32([0]))
    assert got[1].tolist() == [67, 68] and got[4].tolist() == [0] and qlinear.device_error() == 0


def test_rows_of_a_wider_table():
    wide = torch.full((3, 90), 5, **I32)
    view = wide[:, 10:14]
    qlinear.plan_step(view, i32([0, 0, 0]), i32([17, 1, 40]), page_size=16, max_tokens=58, free_pages=i32([9, 8, 7, 6, 4, 3]), taken=i32([0]))
    want = torch.full((3, 90), 5, **I32)
    want[0, 10:12], want[1, 10], want[2, 10:13] = i32([9, 8]), 7, i32([6, 4, 3])
    assert torch.equal(wide, want) and qlinear.device_error() == 0


@pytest.mark.parametrize("bad", ["pages", "columns", "rows", "negative length", "negative count", "negative taken", "sum"])
def test_a_step_without_room_changes_nothing(bad):
    have, new, free, rows, width, taken = [16, 30], [1, 40], [11, 12, 13, 14], 41, 5, 0
    if bad == "pages":
        taken = 1
    if bad == "columns":
        width = 4
    if bad == "rows":
        rows = 40
    if bad == "negative length":
        have[0] = -1
    if bad == "negative count":
        new[0] = -1
    if bad == "negative taken":
        taken = -1
    if bad == "sum":
        have[1] = 2 ** 31 - 5
    table = i32([[3] + [-1] * (width - 1), [4, 5] + [-1] * (width - 2)])
    before = table.clone()
    assert qlinear.device_error() == 0
    got = qlinear.plan_step(table, i32(have), i32(new), page_size=16, max_tokens=rows, free_pages=i32(free), taken=i32([taken]))
    assert qlinear.device_error() == _lib.DEV_ERR_NO_ROOM
    assert got[0].tolist() == [0] * rows and got[1].tolist() == [-1] * rows and got[2].tolist() == [0, 0, 0] and got[3].tolist() == have
    assert got[4].tolist() == [taken] and torch.equal(table, before)


def test_a_page_that_is_not_there_is_reported():
    got = qlinear.plan_step(i32([[3, -1, 5]]), i32([15]), i32([18]), page_size=16, max_tokens=18)
    assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX
    assert got[1].tolist() == [63] + [-1] * 16 + [80] and got[0].tolist() == list(range(15, 33))


@pytest.mark.parametrize("B,new", [(3, [1, 1, 1]), (5, [700, 0, 900, 1, 2500])])
def test_replays_advance_the_sequences(B, new):
    """lengths and taken updated in place by a captured call, one CTA and several; then the same on another
    stream."""
    ps, steps = 16, 5
    have = [7 * b for b in range(B)]
    held = [-(-h // ps) for h in have]
    width = -(-(max(have) + steps * max(new)) // ps)
    free = list(range(5000, 5000 + sum(-(-(h + steps * n) // ps) for h, n in zip(have, new))))
    table, at = [], 0
    for n in held:
        table.append(list(range(at, at + n)) + [-1] * (width - n))
        at += n
    t, lengths, counts, pages, taken = i32(table), i32(have), i32(new), i32(free), i32([0])
    rows = sum(new) + 2
    out = (torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.zeros(rows, dtype=torch.int64, device="cuda"), i32([0] * (B + 1)),
           lengths, taken)
    plan = lambda: qlinear.plan_step(t, lengths, counts, page_size=ps, max_tokens=rows, free_pages=pages, taken=taken, out=out)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # captured, not run
        got = plan()
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(got, out))
    side, used = torch.cuda.Stream(), 0
    for step in range(steps):
        want, table = lists(table, have, new, ps, rows, free, used)
        have, used = want[3], want[4]
        if step % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                plan()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
        assert [o.tolist() for o in out] == [*want[:4], [used]] and t.tolist() == table
    assert qlinear.device_error() == 0


def test_refusals(dev):
    ok = dict(page_table=i32([[1, 2]]), lengths=i32([3]), new_tokens=i32([1]), page_size=16, max_tokens=1, free_pages=i32([4]), taken=i32([0]))
    out = qlinear.plan_step(**ok)
    for bad in (dict(page_table=i32([1, 2])), dict(page_table=i32([[1], [2]])), dict(page_table=ok["page_table"].long()),
                dict(page_table=torch.zeros(4, 2, **I32).t()[:1]), dict(page_table=ok["page_table"].cpu()), dict(lengths=ok["lengths"].long()),
                dict(lengths=ok["lengths"].cpu()), dict(new_tokens=i32([1, 2])), dict(new_tokens=None), dict(max_tokens=-1),
                dict(max_tokens=1 << 31), dict(taken=None), dict(free_pages=None), dict(taken=i32([0, 0])), dict(free_pages=i32([[4]])),
                dict(page_size=1 << 40), dict(out=list(out)), dict(out=out[:4]), dict(out=(out[0].int(), *out[1:])),
                dict(out=(*out[:3], i32([1, 2]), out[4])), dict(page_table=i32([[1, 2]]).expand(2, 2), lengths=i32([1, 1]), new_tokens=i32([0, 0]))):
        with pytest.raises((ValueError, TypeError)):
            qlinear.plan_step(**{**ok, **bad})
    for ps in (0, 12, -16):
        with pytest.raises(qlinear.QlError):
            qlinear.plan_step(**{**ok, "page_size": ps})
    assert qlinear.device_error() == 0

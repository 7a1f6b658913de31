"""CPU: what ql_plan_step_within refuses before any launch."""
import ctypes as C

import pytest

from qlinear import _lib

PAGE = 0x1000000  # addresses far apart
BASE = dict(table=1, stride=8, width=8, lengths=2, new=3, B=2, ps=16, T=4, max_kv=100, free=4, num_free=3, taken=5, positions=6, slots=7, starts=8,
            lens=9, taken_out=10)
WORDS = ("table", "lengths", "new", "free", "taken", "positions", "slots", "starts", "lens", "taken_out")


def call(**kw):
    a = {**{k: v * PAGE if k in WORDS else v for k, v in BASE.items()}, **kw}
    return _lib.lib().ql_plan_step_within(*(C.c_void_p(v) if k in WORDS else v for k, v in a.items()), None)


@pytest.mark.parametrize("max_kv", [-1, 1 << 31])
def test_bound_of_the_lengths(max_kv):
    assert call(max_kv=max_kv) == _lib.QL_EINVAL_SHAPE


def test_the_rest_is_refused_as_without_a_bound():
    for kw in (dict(B=-1), dict(T=-1), dict(T=1 << 31), dict(num_free=-1), dict(stride=7), dict(width=-1)):
        assert call(**kw) == _lib.QL_EINVAL_SHAPE, kw
    for kw in (dict(table=0), dict(lengths=0), dict(new=0), dict(lens=0), dict(starts=0), dict(positions=0), dict(slots=0), dict(taken=0), dict(taken_out=0),
               dict(table=PAGE + 1), dict(slots=PAGE + 4)):
        assert call(**kw) == _lib.QL_EINVAL_ARG, kw
    assert call(ps=12) == _lib.QL_EUNSUPPORTED


def at(name, offset=0):
    return BASE[name] * PAGE + offset


@pytest.mark.parametrize("kw", [
    # an output over an input, whole or in part
    dict(lens=at("new")), dict(lens=at("new", 4)), dict(lens=at("lengths", 4)), dict(lens=at("lengths", -4)), dict(starts=at("lengths")),
    dict(starts=at("new", -8)), dict(starts=at("lengths", -8)), dict(positions=at("lengths")), dict(slots=at("new")), dict(lens=at("free", 8)),
    dict(taken_out=at("lengths", 4)), dict(taken_out=at("free")), dict(taken_out=at("new")), dict(lens=at("taken")), dict(slots=at("free", 8)),
    # over another output
    dict(slots=at("positions")), dict(slots=at("positions", 24)), dict(starts=at("lens", 4)), dict(lens=at("starts", 8)), dict(taken_out=at("starts", 8)),
    dict(lens=at("slots", 28)), dict(lengths=at("lens"), taken_out=at("lens"), B=1),
    # over the page table's rows, which are written too
    dict(positions=at("table")), dict(lens=at("table", 60)), dict(starts=at("table", -8)), dict(lengths=at("table", 28)), dict(free=at("table", 32)),
    dict(taken=at("table", 63 - 3), taken_out=at("table", 63 - 3)), dict(new=at("table", 40), stride=10), dict(lens=at("table", 200), B=7),
], ids=str)
def test_outputs_over_other_arguments(kw):
    assert call(**kw) == _lib.QL_EINVAL_ARG, kw
    assert b"overlaps" in _lib.lib().ql_last_error()

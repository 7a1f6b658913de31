"""GPU: the outputs of a planned step that may lie over its inputs, or between them."""
import pytest
import torch

import qlinear

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_arguments_between_the_rows_of_a_wide_table():
    """Rows of 3 entries, 8 apart; lengths, counts and the outputs of int32 in the gaps."""
    wide = torch.full((4, 8), 9, dtype=torch.int32, device="cuda")
    table, lengths, new, lens = wide[:2, :3], wide[0, 3:5], wide[0, 5:7], wide[1, 3:5]
    starts, taken, taken_out = wide[1, 5:8], wide[2, 0:1], wide[2, 1:2]
    lengths.copy_(i32([0, 16])), new.copy_(i32([2, 1])), taken.zero_()
    table[1, 0] = 4
    out = (torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), starts, lens, taken_out)
    qlinear.plan_step(table, lengths, new, page_size=16, max_tokens=3, free_pages=i32([7, 5]), taken=taken, out=out)
    assert out[0].tolist() == [0, 1, 16] and out[1].tolist() == [112, 113, 80]
    assert wide.tolist() == [[7, 9, 9, 0, 16, 2, 1, 9], [4, 5, 9, 2, 17, 0, 2, 3], [0, 2, 9, 9, 9, 9, 9, 9], [9] * 8]
    assert qlinear.device_error() == 0


@pytest.mark.parametrize("name", ["new_tokens", "q_starts", "free_pages"])
def test_lengths_over_something_else_are_refused(name):
    a = dict(page_table=i32([[1, -1], [2, -1]]), lengths=i32([3, 16]), new_tokens=i32([1, 1]), page_size=16, max_tokens=2, free_pages=i32([4, 5]),
             taken=i32([0]))
    out = list(qlinear.plan_step(**a))
    out[3] = a[name] if name in a else out[2][:2]
    with pytest.raises(qlinear.QlError):
        qlinear.plan_step(**a, out=tuple(out))
    assert qlinear.device_error() == 0

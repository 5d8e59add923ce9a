"""A step count in memory that the same AdamW step writes: workgroups that start late would take another step."""
import pytest

from test_block_layers import F16, F32, I64, U8, adamw, at, errors, one


def inside(place, offset):
    t = at(place, (1,), I64)
    t.data += offset
    return t


# what lies there: parameter 0, m 2, v 3, m's scales 4, v's scales 5, master copy 6 (`one`), an array's first bytes, its last and, of four bytes, its end and the one before
@pytest.mark.parametrize('place,offset', [(0, 0), (0, 3992), (0, 3996), (0, -4), (2, 0), (2, 2000), (3, 3996)])
def test_adamw_refuses_a_step_count_in_what_it_writes(place, offset):
    adamw(errors()[0], [one()], t_array=inside(place, offset))
    adamw(errors()[0], [one(place=10), one()], t_array=inside(place, offset))


def test_adamw_refuses_a_step_count_among_scales_codes_and_master_copies():
    for place, offset in ((2, 992), (3, 0), (4, 8), (5, 12)):
        adamw(errors()[0], [one(8)], t_array=inside(place, offset))
    for place, offset in ((0, 1992), (6, 3992)):
        adamw(errors()[0], [one(dtype=F16, master=at(6, (1000,), F32))], t_array=inside(place, offset))
    assert one(8)[2].dtype == U8

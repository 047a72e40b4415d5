"""zt_kv8_plan's workgroups read what others write if its outputs lie in its
inputs: such calls are refused (nothing is launched: the pointers are not real)."""
import itertools

import pytest

from ztensor_amd import _lib

BAD = _lib.HIP_ERROR_INVALID_VALUE
NAMES = ("lens add table requests width free count capacity page tokens table_out slots positions q_start lens_out "
         "count_out").split()
R, WIDTH, CAPACITY, TOKENS = 4, 8, 16, 9
SIZE = {"lens": 4 * R, "add": 4 * R, "table": 4 * R * WIDTH, "free": 4 * CAPACITY, "count": 4, "table_out": 4 * R * WIDTH,
        "slots": 8 * TOKENS, "positions": 4 * TOKENS, "q_start": 4 * R + 4, "lens_out": 4 * R, "count_out": 4}
INPUTS, OUTPUTS = ("lens", "add", "table", "free", "count"), ("table_out", "slots", "positions", "q_start", "lens_out", "count_out")


def call(**other):
    good = {n: (1 << 20) + 4096 * i for i, n in enumerate(SIZE)}
    good.update(requests=R, width=WIDTH, capacity=CAPACITY, page=16, tokens=TOKENS)
    return _lib.load().zt_kv8_plan(*({**good, **other}[n] for n in NAMES), None)


@pytest.mark.parametrize("out,other", [(a, b) for a, b in itertools.product(OUTPUTS, INPUTS + OUTPUTS) if a != b])
def test_overlaps_are_refused(out, other):
    at, step = 1 << 24, 8 if "slots" in (out, other) else 4
    if (out, other) != ("table_out", "table"):  # a table may be written in place
        assert call(**{out: at, other: at}) == BAD
    assert call(**{out: at, other: at + (SIZE[out] - 1) // step * step}) == BAD or SIZE[out] <= step
    assert call(**{out: at + (SIZE[other] - 1) // step * step, other: at}) == BAD or SIZE[other] <= step

"""Borders of the token mixers' host arithmetic: no GPU."""
import ctypes
import random

import pytest


def deal_bounds(dh, total, slots, pairs, least=4):
    lo, hi = ctypes.c_int32(), ctypes.c_int32()
    dh.lib.dragon_window_deal_bounds(float(total), slots, pairs, least, ctypes.byref(lo), ctypes.byref(hi))
    return lo.value, hi.value


def parts(steps, longest):
    return sum(max(-(-s // longest), 1) for s in steps)


@pytest.mark.parametrize("pairs", (1, 2, 3, 60, 256, 500, 505, 508, 510, 511, 512))
@pytest.mark.parametrize("most", (1, 100, 70000, 1 << 22, 1 << 25))
def test_the_parts_fit_the_slots_at_the_upper_bound(dh, pairs, most):
    """512 slots; a tile has up to 2^25 steps (2^30 keys, 32 at a time).  With one slot to spare all / (slots - pairs) is the
    sum of all steps, up to 2^34."""
    rng = random.Random(pairs * 31 + most)
    for steps in ([most] * pairs, [rng.randint(0, most) for _ in range(pairs)], [most] + [0] * (pairs - 1)):
        lo, hi = deal_bounds(dh, sum(steps), 512, pairs)
        assert 4 <= lo <= hi
        assert parts(steps, hi) <= 512
        assert lo == 4 or parts(steps, lo - 1) > 512        # what lies below lo does not fit

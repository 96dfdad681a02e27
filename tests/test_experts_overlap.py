"""Calls that would write what they still have to read are refused; columns side by side in one buffer are not (no GPU needed)."""
import ctypes as C
import random

import pytest

import iree_b200 as ib
from iree_b200.runtime import library

BASE = 1 << 20
TABLE = 1 << 30


def overlaps(name, params, *args):
    """Whether the call refuses its arrays for that reason, and not just for the missing context."""
    assert getattr(library(), "iree_b200_" + name)(None, C.addressof(params), *args) == 3
    message = library().iree_b200_last_error().decode()
    assert ("overlap" in message) != ("context" in message), message
    return "overlap" in message


def calls(params, token_side, row_side):
    """Every call with a result and an input of those two addresses."""
    t = TABLE
    return [overlaps("expert_dispatch", params, t, token_side, t, t, t, row_side, None),
            overlaps("expert_dispatch_backward", params, row_side, t, token_side),
            overlaps("expert_combine", params, row_side, t, t, token_side),
            overlaps("expert_combine_backward", params, token_side, BASE << 8, t, t, row_side, t)]


def elements(address, rows, width, pitch):
    return {address + 2 * (r * pitch + c) for r in range(rows) for c in range(width)}


def test_against_the_elements_themselves(built):
    """Arrays of one pitch, or without gaps, or of one row: refused exactly where they share an element."""
    rng = random.Random(7)
    seen = set()
    for _ in range(1500):
        T, k, width = rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 6)
        kind = rng.randint(0, 2)
        tp = rp = width + rng.choice([0, 1, width, 2 * width + 3])
        if kind == 1:
            tp = rp = width
        elif kind == 2:
            T, tp = 1, rng.randint(width, 3 * width)
        p = ib.ExpertRowsParams(ib.KIND_F16, T, k, 4, 0, width, tp, rp)
        x, rows = BASE, BASE + 2 * rng.randint(-60, 60)
        want = bool(elements(x, T, width, tp) & elements(rows, T * k, width, rp))
        assert calls(p, x, rows) == [want] * 4, (T, k, width, tp, rp, rows - x)
        seen.add((kind, want))
    assert len(seen) == 6


def test_gradients_of_rows_against_rows(built):
    T, k, width = 5, 2, 16
    p = ib.ExpertRowsParams(ib.KIND_BF16, T, k, 4, 0, width, width, 2 * width)
    dout, t, rows = BASE << 8, TABLE, BASE
    last = 2 * ((T * k - 1) * 2 * width)
    for shift, want in ((0, True), (2 * width, False), (2 * (width - 1), True), (2 * (width + 1), True), (last, True), (last + 2 * width, False),
                        (-last, True), (-2 * width, False)):
        assert overlaps("expert_combine_backward", p, dout, rows, t, t, rows + shift, t) == want, shift


@pytest.mark.parametrize("T, width", [(0, 16), (4, 0)])
def test_empty_arrays_share_nothing(built, T, width):
    p = ib.ExpertRowsParams(ib.KIND_F16, T, 2, 4, 0, width, 16, 16)
    assert calls(p, BASE, BASE) == [False] * 4

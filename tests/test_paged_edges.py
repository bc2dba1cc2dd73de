"""The paged operators on the host (no device), at the edges of what a call may
hold: rows beyond the step's, refusals."""
import ctypes as C

import pytest

import infer_hip as H
import oracle_lib as O
from test_paged import A, attention, pages, qkrope, refused


def row(first, end, rows):
    f = O.lib().orc_paged_row
    f.restype = C.c_int32
    f.argtypes = [C.c_int32, C.c_int32, C.c_int32]
    return f(first, end, rows)


@pytest.mark.parametrize("rows", [1, 2, 7, 2 ** 31 - 1])
def test_rows_stay_in_the_step(rows):
    """A sequence's row is the last of its own, and never one that the arrays do not have."""
    low, high = -2 ** 31, 2 ** 31 - 1
    for first in (low, -1, 0, 1, 5, 6, high - 1, high):
        for end in (low, -1, 0, 1, 2, 6, 7, 8, high):
            r = row(first, end, rows)
            assert r == (end - 1 if end > first and 1 <= end <= rows else -1), (first, end)
            assert -1 <= r < rows


def test_rows_without_offsets():
    """Row s of sequence s, where there is one."""
    assert [row(s, s + 1, 3) for s in range(6)] == [0, 1, 2, -1, -1, -1]


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("scale", [-0.125, -1e-300, 1e39, 3e38])
def test_attention_scales_refused(scale):
    """A scale below 0 (which no formula here has: 0 alone stands for the default), and one that
    leaves single when the exponential's base is 2."""
    refused(lambda: attention(pages(), scale=scale), -1, "scale")


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-30, 2.3e38])
def test_attention_scales_taken(scale):
    refused(lambda: attention(pages(), scale=scale), -1, "no context")


@pytest.mark.parametrize("skew", [1, 2, 3])
def test_unaligned_numbers_refused(skew):
    """Lengths, tables, positions and slots are int32, aligned to 4 bytes, as the attention's are."""
    names = ("past", "count", "seqs", "table", "max_pages", "page_size", "ring", "pages", "ends", "ends_out", "offsets",
             "lengths", "positions", "slots", "rows", "failed")
    good = dict(zip(names, (A, A, 3, A, 4, 16, A, 9, A, A, A, A, A, A, 7, A)))

    def slots(**kw):
        return H.lib().ihip_enqueue_paged_slots(None, *dict(good, **kw).values())

    refused(slots, -1, "no context")
    for name in ("past", "count", "table", "ring", "offsets", "lengths", "positions", "slots", "failed"):
        refused(lambda: slots(**{name: A + skew}), -1, "4 bytes")
    for name in ("positions", "slots"):
        refused(lambda: qkrope(pages(), **{name: A + skew}), -1, "4 bytes")

"""Draws of rows whose first or last tokens cannot be drawn (constrained decoding), and of more
rows with bins than one launch has places for, against the definition in 64 bits."""
import numpy as np
import pytest

import sample_ref as S
from test_gpu_paged import ctx, dev  # noqa: F401 (fixtures)
from test_gpu_sample_rows import MIXED, Rows, zipf

pytestmark = pytest.mark.gpu
FREE = (1.0, 0, 1.0, 0.0)
LAST = 1 - 2.0 ** -53


@pytest.mark.parametrize("rows", [8, 600, 1200])  # (parts of 2048, 4096 and 8192 tokens)
def test_the_ends_of_a_row_are_masked(ctx, dev, rows):
    """0 draws the first token that has a weight, though whole groups of tokens before it have none,
    and the largest number below 1 the last one, whose weight here is the row's largest (so that no
    rounding of the sums reaches past it)."""
    rng = np.random.default_rng(rows)
    vocab = 20011
    x, u, want = zipf(rng, rows, vocab), np.zeros(rows), np.zeros(rows, int)
    for r in range(rows):
        head, tail = [(512, 0), (1024, 512), (700, 1), (8192 + 512, 600), (512 * 37, 0), (4095, 1025), (0, 512), (1, 9000)][r % 8]
        none = -np.inf if r // 8 % 2 == 0 else np.nan
        x[r, :head], x[r, vocab - tail:] = none, none
        last = vocab - tail - 1
        x[r, last] = 30
        u[r] = 0 if rng.random() < 0.7 else LAST
        want[r] = head if u[r] == 0 else last
        assert S.draw(x[r], *FREE, u[r])[0] == want[r]
    b = Rows(dev, x, [FREE] * rows, u)
    b.enqueue(ctx)
    ids, probs = b.read()
    assert np.array_equal(ids, want), np.argwhere(ids != want)[:8].ravel()
    p = np.array([S.draw(x[r], *FREE, u[r])[1] for r in range(rows)])
    assert (np.abs(probs - p) <= p * (2.0 ** -24 + 1e-9) + 1e-30).all()


def test_masked_groups_within_a_row(ctx, dev):
    """Any number, with whole groups and parts of the row masked, behind either end and between."""
    rng = np.random.default_rng(5)
    vocab, rows = 30000, 64
    x = zipf(rng, rows, vocab)
    for r in range(rows):
        for i in range(0, vocab, 512):
            if rng.random() < [0.2, 0.5, 0.9][r % 3]:
                x[r, i:i + 512] = -np.inf if rng.random() < 0.5 else np.nan
        x[r, rng.integers(0, vocab)] = 3
    Rows(dev, x, [FREE, MIXED[5], MIXED[6], (0.3, 0, 1.0, 0.0)] * (rows // 4), rng.random(rows)).check(ctx)


def test_weights_that_are_none(ctx, dev):
    """Tokens below 2^-1000 of the best one's weight are none, also where they stand before others
    of a part whose own best is that small: 0 draws the first one above."""
    vocab = 9000
    x = np.full((3, vocab), -720.0, np.float32)  # 2^-1039
    x[0, 1500], x[0, 1700], x[0, 4000] = -350, -690, 0
    x[1, 1500], x[1, 8999] = -692, 0  # 2^-998
    x[2, 2047], x[2, 2048] = -694, 0  # 2^-1001
    b = Rows(dev, x, [FREE] * 3, np.zeros(3))
    b.enqueue(ctx)
    ids, probs = b.read()
    assert ids.tolist() == [1500, 1500, 2048]
    assert probs[2] == 1


def test_more_rows_with_bins_than_places(ctx, dev):
    """Every row has more candidates than are sorted; 512 of a launch have bins formed by the whole
    grid, which ones by chance, and the others form theirs alone: all the same, from run to run,
    and the next call's are counted from 0 again."""
    rng = np.random.default_rng(6)
    rows, vocab = 620, 5003
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    b = Rows(dev, x, [(30.0, 0, 0.5, 0.0)] * rows, rng.random(rows))
    b.check(ctx)
    ids, probs = b.read()
    for _ in range(2):
        b.enqueue(ctx)
        again = b.read()
        assert np.array_equal(again[0], ids) and np.array_equal(again[1].view(np.uint32), probs.view(np.uint32))
    few = Rows(dev, x[:5], [(30.0, 0, 0.5, 0.0)] * 5, b.u[:5])
    few.check(ctx)
    assert np.array_equal(few.read()[0], ids[:5])

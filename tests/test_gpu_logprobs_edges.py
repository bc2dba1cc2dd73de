"""ihip_enqueue_logprobs at its largest sizes, against paged_ref.py."""
import numpy as np
import pytest

from test_gpu_logprobs import check, ctx, logits  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def test_logprobs_rows_beyond_a_launch(ctx):
    """More rows than a grid's second dimension holds: the outputs of the second launch follow."""
    rng = np.random.default_rng(1)
    rows = 65535 + 700
    check(ctx, logits(rng, rows, 37), rng.integers(0, 37, rows), 3)


@pytest.mark.parametrize("k", [0, 1, 64])
def test_logprobs_largest_vocabulary(ctx, k):
    rng = np.random.default_rng(2)
    x = logits(rng, 2, 1 << 22)
    x[1, -5:] = 30
    check(ctx, x, np.array([(1 << 22) - 1, (1 << 22) - 3]), k)

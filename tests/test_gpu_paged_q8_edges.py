"""8-bit pages on the device: one key whose value scale is far above the others', and whose weight is
next to nothing, against the definition in 64 bits."""
import numpy as np
import pytest

from test_gpu_paged import ctx, dev  # noqa: F401 (fixtures)
from test_gpu_paged_q8 import Batch
from test_gpu_paged_shared import Batch as Groups

pytestmark = pytest.mark.gpu


def outlier(page, at, codes, scales, ratio):
    """Token `at` of the page: a score of -60 and less for queries of positive values, and values
    `ratio` times as large."""
    codes[0][page, at], scales[0][page, at] = -127, 1.0
    scales[1][page, at] *= ratio


@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 20, 2.0 ** 30])
@pytest.mark.parametrize("at", [0, 40, 299])
@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 16, 2), (256, 4, 1), (512, 4, 1), (96, 6, 3)])
def test_a_value_scale_far_above_the_others(ctx, dev, hd, heads, kvh, at, ratio):
    """What a weight may lose is 2^-39 of the largest scale (Batch.want), whatever that one's key
    weighs: the other keys keep all bits of single up to scales 2^15 apart, 9 of them at 2^30."""
    b = Batch(np.random.default_rng(at), hd, heads, kvh, 16, [300, 300], spread=0.0)
    b.q = np.abs(b.q) + np.float32(0.1)
    outlier(b.table[0, at // 16], at % 16, b.codes, b.scales, ratio)
    b.check(ctx, dev)


@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 20, 2.0 ** 30])
@pytest.mark.parametrize("at", [0, 250, 310])
@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 16, 2), (256, 4, 1)])
def test_in_a_group(ctx, dev, hd, heads, kvh, at, ratio):
    """The same of a prefix and of own tokens."""
    b = Groups(np.random.default_rng(at), "q8", hd, heads, kvh, 16, [(5, 288, 288)], [320, 300, 288, 330, 319])
    b.q = np.abs(b.q) + np.float32(0.1)
    outlier(b.table[0, at // 16], at % 16, b.raw[:2], b.raw[2:], ratio)
    b.check(ctx, dev)

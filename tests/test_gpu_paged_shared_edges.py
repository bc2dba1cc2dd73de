"""Attention of groups that share their first tokens, beside that without groups: large scores and
sinks that are infinite, for prefixes that one block finishes and that blocks share."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_ref as R
from test_gpu_paged import assert_close, ctx, dev  # noqa: F401 (fixtures)
from test_gpu_paged_shared import DTYPES, Batch

pytestmark = pytest.mark.gpu


def alone(ctx, dev, b):
    """The same call without its groups."""
    y = dev.out(b.q.nbytes)
    H.check(H.lib().ihip_enqueue_paged_attention(ctx.h, b.dq, 0, C.byref(b.pool), b.dt, b.width, b.dl, y.ptr, len(b.q), b.heads,
                                                 0, b.ds, b.scale), "attention")
    return y.download(np.float32, b.q.size).reshape(b.q.shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("prefix", [30, 1900])
def test_large_scores_of_all_keys(ctx, dev, dtype, hd, prefix):
    """All keys of a head have one score, of up to 2000 in base 2, so that all weights are 1 whatever
    the score was rounded to. Values are 1 in the prefix and -1 behind it: sums of whole numbers
    below 2^24, which single holds, and their quotient, a rounding (2 U of the result here)."""
    rng = np.random.default_rng(hd + prefix)
    heads, kvh, ps = 8, 2, 16
    own = [0, 1, 7, 29, 100, prefix // 2, prefix]
    b = Batch(rng, dtype, hd, heads, kvh, ps, [(len(own), prefix, -(-prefix // ps) * ps)], [prefix + o for o in own])
    scale, code = (2.0 ** -6, 64) if dtype == "q8" else (1.0, 1)
    k, v = b.raw[:2]
    k[...] = 0
    k[..., 3] = (100 if dtype == "q8" else R.pack(np.array([6.25]), dtype)[0])
    one = np.array([code]) if dtype == "q8" else R.pack(np.array([1.0]), dtype)
    less = np.array([-code]) if dtype == "q8" else R.pack(np.array([-1.0]), dtype)
    v[...] = less[0]
    for p, t in R.keys_of(b.table[0], prefix, 0, ps, b.pages):
        v[p, t] = one[0]
    # (a page that is not full when the sequences part: each has the prefix's tokens in its own copy)
    for s in range(len(own)):
        for p, t in R.keys_of(b.table[s], prefix, 0, ps, b.pages):
            v[p, t] = one[0]
    if dtype == "q8":
        b.raw[2][...], b.raw[3][...] = 0.0625, scale
    b.q[...] = 0
    b.q[..., 3] = np.array([3.0, 37.0, 111.0, 150.0, 171.0, 199.0, 211.0, 221.0], np.float32)
    b.scale = 1.0
    b.upload(dev)
    b.enqueue(ctx)
    got = b.read()
    want = np.array([(prefix - o) / (prefix + o) for o in own])[:, None, None] * np.ones_like(got)
    assert_close(got, want, 2 * R.U * np.abs(want) + 1e-12)
    assert_close(alone(ctx, dev, b), want, 2 * R.U * np.abs(want) + 1e-12)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix", [30, 1900])
def test_sinks_of_infinity(ctx, dev, dtype, prefix):
    """A sink of +infinity, or one that its scaling makes so, has all of the weight, one of -infinity
    none, a NaN is one: in a group as without it. A sequence without a key gives zeros."""
    rng = np.random.default_rng(prefix)
    b = Batch(rng, dtype, 128, 8, 2, 16, [(6, prefix, -(-prefix // 16) * 16)],
              [prefix, prefix + 1, prefix + 40, 5, 0, prefix + 300], alone=2, behind=1)
    b.lengths[0] = 0  # (outside the group too)
    big = np.finfo(np.float32).max
    b.sinks = np.array([np.inf, -np.inf, 0.5, big, -big, np.nan, -2.0, 1.0], np.float32)
    b.upload(dev)
    b.enqueue(ctx)
    got, without = b.read(), alone(ctx, dev, b)
    off = b.sinks.copy()
    off[[0, 3, 4, 5]] = -np.inf
    b.sinks = off
    want, tol = b.want()
    want[:, [0, 3]], tol[:, [0, 3]] = 0, 0
    live = b.lengths > 0
    ok = [0, 1, 2, 3, 4, 6, 7]
    for y in (got, without):
        assert_close(y[:, ok], want[:, ok], tol[:, ok])
        assert np.isnan(y[live, 5]).all() and (y[b.lengths == 0] == 0).all()

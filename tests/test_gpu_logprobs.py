"""ihip_enqueue_logprobs on the device against the definition in 64 bits
(paged_ref.py)."""
import numpy as np
import pytest

import infer_hip as H
import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = H.Context(0)
    yield c
    c.close()


def run(ctx, x, ids, k, pad=0, skew=0, entropy=True):
    rows, vocab = x.shape
    wide = np.full((rows, vocab + pad), np.nan, np.float32)
    wide[:, :vocab] = x
    buf = ctx.alloc(wide.nbytes + 4 * skew)
    H.check(H.lib().ihip_upload(ctx.h, buf.ptr + 4 * skew, H._p(wide), wide.nbytes))
    bufs = [buf] + [ctx.array(np.full(max(n, 1) + 1, -77, np.int32)) for n in (rows, rows, rows * k, rows * k)]
    di = ctx.array(ids.astype(np.int32)) if ids is not None else None
    _, lp, ent, ti, tl = bufs
    H.check(H.lib().ihip_enqueue_logprobs(
        ctx.h, buf.ptr + 4 * skew, rows, vocab, vocab + pad if pad else 0, di.ptr if di else 0,
        lp.ptr if di else 0, ent.ptr if entropy else 0, k, ti.ptr if k else 0, tl.ptr if k else 0), "logprobs")
    out = (lp.download(np.float32, rows), ent.download(np.float32, rows),
           ti.download(np.int32, rows * k).reshape(rows, k), tl.download(np.float32, rows * k).reshape(rows, k))
    for b, n in ((lp, rows), (ent, rows), (ti, rows * k), (tl, rows * k)):
        assert b.download(np.int32, n + 1)[n] == -77
    for b in bufs + ([di] if di else []):
        b.free()
    return out


def check(ctx, x, ids, k, **kw):
    got = run(ctx, x, ids, k, **kw)
    with np.errstate(divide="ignore", invalid="ignore"):
        lp, ent, top_ids, top, t_lp, t_ent, t_top = R.logprobs(x, ids, k)
    assert np.array_equal(got[2], top_ids)
    for g, w, t in ((got[0], lp, t_lp), (got[1], ent, t_ent), (got[3], top, t_top)):
        if g is got[0] and ids is None:
            continue
        fine = np.isfinite(w)
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)])
        assert np.all(np.abs(g[fine] - w[fine]) <= t[fine]), (np.abs(g[fine] - w[fine]).max(), t[fine].min())


def logits(rng, rows, vocab, sharp=2.5):
    x = (rng.standard_normal((rows, vocab)) * sharp).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 12
    return x


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 256, 1000, 4095, 4097, 16384, 32000, 151936])
@pytest.mark.parametrize("rows,k", [(1, 20), (3, 0), (5, 1), (2, 64), (7, 5)])
def test_logprobs(ctx, vocab, rows, k):
    rng = np.random.default_rng(vocab + k)
    x = logits(rng, rows, vocab)
    check(ctx, x, rng.integers(0, vocab, rows), k)


@pytest.mark.parametrize("rows,vocab,k", [(300, 5000, 3), (1030, 700, 20), (64, 40000, 8)])
def test_logprobs_many_rows(ctx, rows, vocab, k):
    rng = np.random.default_rng(rows)
    check(ctx, logits(rng, rows, vocab), rng.integers(0, vocab, rows), k)


@pytest.mark.parametrize("pad,skew", [(0, 1), (1, 0), (3, 2), (5, 3), (4, 0), (64, 1)])
def test_logprobs_strides_and_alignment(ctx, pad, skew):
    rng = np.random.default_rng(pad * 7 + skew)
    for vocab in (999, 20001, 66):
        check(ctx, logits(rng, 4, vocab), rng.integers(0, vocab, 4), 9, pad=pad, skew=skew)


def test_logprobs_ties(ctx):
    """Equal logits: the lowest ids first, whole rows of them, in blocks, and both zeros."""
    rng = np.random.default_rng(3)
    x = np.zeros((6, 30000), np.float32)
    x[1] = rng.integers(0, 3, 30000)
    x[2] = rng.integers(0, 2000, 30000) / 64
    x[3, ::2] = -0.0
    x[4, 12345:] = 1
    x[5, 29990:] = 1
    for k in (1, 7, 64):
        check(ctx, x, rng.integers(0, 30000, 6), k)


def test_logprobs_masked(ctx):
    """-infinity and the type's lowest value: few allowed tokens, one, none."""
    rng = np.random.default_rng(4)
    x = np.full((7, 50000), -np.inf, np.float32)
    at = rng.integers(0, 50000, 5)
    x[0, at] = rng.standard_normal(5)
    x[1, 49999] = -3e38
    x[3] = np.finfo(np.float32).min
    x[4] = np.finfo(np.float32).min
    x[4, at] = rng.standard_normal(5)
    x[5] = logits(rng, 1, 50000)[0]
    x[5, ::2] = -np.inf
    x[6, :] = np.float32(3e38)
    ids = np.array([at[0], 49999, 3, 17, at[1], 2, 9])
    for k in (1, 20, 64):
        check(ctx, x, ids, k)


def test_logprobs_nan_and_infinity(ctx):
    rng = np.random.default_rng(5)
    x = logits(rng, 6, 9000)
    x[0, 77] = np.nan
    x[1] = np.nan
    x[2, 5] = np.inf
    x[3, [8, 4000]] = np.inf
    x[4, ::3] = np.nan
    # the rows beside them are as they are alone
    check(ctx, x, rng.integers(0, 9000, 6), 20)
    check(ctx, x[:, :30], rng.integers(0, 30, 6), 40)


def test_logprobs_ids_outside(ctx):
    rng = np.random.default_rng(6)
    ids = np.array([-1, 5000, 4999, 0, 2 ** 31 - 1, -2 ** 31])
    check(ctx, logits(rng, 6, 5000), ids, 2)
    assert np.isnan(run(ctx, logits(rng, 6, 5000), ids, 2)[0]).tolist() == [True, True, False, False, True, True]


def test_logprobs_parts(ctx):
    """Only the alternatives, only the entropy, only the given tokens."""
    rng = np.random.default_rng(7)
    x = logits(rng, 3, 7000)
    check(ctx, x, None, 4)
    a = run(ctx, x, None, 0)
    b = run(ctx, x, rng.integers(0, 7000, 3), 4)
    assert np.array_equal(a[1], b[1])
    c = run(ctx, x, rng.integers(0, 7000, 3), 0, entropy=False)
    assert np.isfinite(c[0]).all() and (c[1].view(np.int32) == -77).all()


def test_logprobs_sharp(ctx):
    """Rows whose one token has nearly all the weight: the entropy's small values."""
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((5, 20000)) * 2).astype(np.float32)
    for r, top in enumerate((20, 40, 80, 200, 1e4)):
        x[r, 1000 * r + 7] = top
    check(ctx, x, np.array([7, 1007, 5, 3007, 4007]), 20)


def test_logprobs_captured(ctx):
    """One graph replayed over other logits, eager calls of another size between the replays."""
    rng = np.random.default_rng(9)
    rows, vocab, k = 4, 33000, 6
    x = logits(rng, rows, vocab)
    dx, di = ctx.array(x), ctx.array(np.zeros(rows, np.int32))
    o = [ctx.alloc(4 * rows * m) for m in (1, 1, k, k)]

    def call():
        H.check(H.lib().ihip_enqueue_logprobs(ctx.h, dx.ptr, rows, vocab, 0, di.ptr, o[0].ptr, o[1].ptr, k, o[2].ptr,
                                              o[3].ptr))

    call()
    H.check(H.lib().ihip_capture_begin(ctx.h))
    call()
    H.check(H.lib().ihip_capture_end(ctx.h, 11))
    for i in range(4):
        x, ids = logits(rng, rows, vocab), rng.integers(0, vocab, rows).astype(np.int32)
        dx.upload(x), di.upload(ids)
        H.check(H.lib().ihip_graph_launch(ctx.h, 11))
        got = [b.download(np.float32, rows * m) for b, m in zip(o, (1, 1, k, k))]
        want = run(ctx, x, ids, k)
        for g, w in zip(got, want):
            assert np.array_equal(g.view(np.int32), w.ravel().view(np.int32))
        check(ctx, logits(rng, 90, 2000), rng.integers(0, 2000, 90), 3)
    for b in [dx, di] + o:
        b.free()

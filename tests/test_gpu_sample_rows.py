"""Draws of many rows on the device against the definition in 64 bits (sample_ref.py) and
the device's own sampler of one row."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import sample_ref as S
from test_gpu_paged import ctx, dev  # noqa: F401 (fixtures)
from test_sample_rows import splitmix

pytestmark = pytest.mark.gpu


def settings_array(rows):
    a = (H.Sampling * len(rows))(*[H.sampling(*r) for r in rows])
    return np.frombuffer(bytes(a), np.uint8).copy()


class Rows:
    def __init__(self, dev, x, settings, u, pad=0, shift=0):
        self.x, self.settings, self.u = x, settings, np.array(u, np.float64)
        rows, vocab = x.shape
        raw = np.full(rows * (vocab + pad) + 8, np.nan, np.float32)
        raw[shift:shift + rows * (vocab + pad)].reshape(rows, vocab + pad)[:, :vocab] = x
        self.args = (dev(raw) + 4 * shift, rows, vocab, vocab + pad if pad else 0, dev(settings_array(settings)), dev(self.u))
        self.ids, self.probs = dev.out(4 * rows + 16), dev.out(4 * rows + 16)

    def enqueue(self, ctx, probs=True):
        H.check(H.lib().ihip_enqueue_sample_rows(ctx.h, *self.args, self.ids.ptr, self.probs.ptr if probs else 0), "sample")

    def read(self):
        n = len(self.x)
        for b in (self.ids, self.probs):
            assert (b.download(np.uint8, 4 * n + 16)[4 * n:] == 0x5A).all()
        return self.ids.download(np.int32, n), self.probs.download(np.float32, n)

    def check(self, ctx, share=0.97, near=1e-10):
        """The definition's ids, but where one of its comparisons is nearer than `near`: weights in
        double are off by 1e-15 of themselves, and by 2^-40 of the best one (2^-61 times the
        vocabulary) where they are whole numbers; up to 2^22 of them over a sum of 1 at least
        2^-22 2^22 2^-39 = 2e-12 as random errors, and what a border is compared with as much. At
        least `share` of the rows are further (none of a kind whose weights are alike)."""
        self.enqueue(ctx)
        ids, probs = self.read()
        far = 0
        for r in range(len(self.x)):
            t, k, p, m = self.settings[r][:4]
            want, prob, margin = S.draw(self.x[r], t, k, p, m, self.u[r])
            if margin < near:
                continue
            far += 1
            assert ids[r] == want, (r, self.settings[r], self.u[r], ids[r], want, margin)
            assert abs(probs[r] - prob) <= prob * (2.0 ** -24 + 1e-9) + 1e-30, (r, self.settings[r], probs[r], prob)
        assert far >= len(self.x) * share - 1
        return ids


def zipf(rng, rows, vocab, least=1.1, most=3.5):
    x = -rng.uniform(least, most, (rows, 1)) * np.log1p(rng.random((rows, vocab)) * vocab) + 18
    return x.astype(np.float32)


MIXED = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 64, 0.95, 0.0),
         (0.8, 0, 0.95, 0.05), (1.0, 0, 0.9, 0.0), (0.8, 40, 1.0, 0.0), (-1.0, 5, 0.5, 0.1), (1e-31, 0, 1.0, 0.0),
         (1e-3, 0, 1.0, 0.0), (5.0, 0, 0.99, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, 1000, 0.999, 0.001),
         (2.0, 0, 1.0, 1e-6), (1.0, 5000, 1.0, 0.0), (1.0, 10 ** 9, 0.7, 0.0), (30.0, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.9)]


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 255, 257, 1025, 2048, 2049, 8195, 50000, 151936, 262149])
@pytest.mark.parametrize("kind", ["zipf", "normal", "flat", "steps"])
def test_settings_by_rows(ctx, dev, vocab, kind):
    rng = np.random.default_rng(vocab)
    n = 2 * len(MIXED)
    if kind == "zipf":
        x = zipf(rng, n, vocab)
    elif kind == "normal":
        x = (rng.standard_normal((n, vocab)) * 2.5).astype(np.float32)
    elif kind == "flat":
        x = np.full((n, vocab), -3.25, np.float32)
    else:  # many ties
        x = np.round(rng.standard_normal((n, vocab)) * 2).astype(np.float32)
    Rows(dev, x, MIXED * 2, rng.random(n)).check(ctx, 0.97 if kind in ("zipf", "normal") else 0.3)


@pytest.mark.parametrize("rows,vocab,pad,shift", [(1, 151936, 0, 0), (3, 32000, 5, 1), (700, 5000, 3, 2), (600, 20011, 0, 0),
                                                  (2, 1 << 22, 0, 0)])
def test_many_rows_strides_and_sizes(ctx, dev, rows, vocab, pad, shift):
    rng = np.random.default_rng(rows)
    x = zipf(rng, rows, vocab)
    Rows(dev, x, [MIXED[(3 * i + 2) % len(MIXED)] for i in range(rows)], rng.random(rows), pad, shift).check(ctx)


def test_rows_behind_a_launch(ctx, dev):
    """More rows than one launch's results find place for."""
    rng = np.random.default_rng(2)
    vocab, rows = 100, 70000
    x = np.tile(zipf(rng, 7, vocab), (10000, 1))
    sets = [MIXED[i % len(MIXED)] for i in range(rows)]
    r = Rows(dev, x, sets, rng.random(rows))
    r.enqueue(ctx)
    ids, _ = r.read()
    for i in [*range(40), *range(65500, 65570), 69998, 69999]:
        t, k, p, m = sets[i]
        want, _, margin = S.draw(x[i], t, k, p, m, r.u[i])
        assert ids[i] == want or margin < 1e-10, i


def test_random_numbers_at_their_ends(ctx, dev):
    """0 draws the first that has a weight, the largest below 1 the last; outside [0, 1) and NaN
    draw a token that is there."""
    rng = np.random.default_rng(3)
    vocab = 9000
    x = zipf(rng, 16, vocab, 1.5, 2)
    x[:, [0, vocab - 1]] = -np.inf
    sets = [(1.0, 0, 1.0, 0.0), (1.0, 7, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (50.0, 0, 0.95, 0.0)] * 4
    u = np.repeat([0.0, 1 - 2.0 ** -53, 1.5, np.nan], 4)
    r = Rows(dev, x, sets, u)
    r.enqueue(ctx)
    ids, probs = r.read()
    for i in range(16):
        s, logits = sets[i], x[i].astype(np.float64)
        by_logit = np.lexsort((np.arange(vocab), -logits))
        assert 0 < ids[i] < vocab - 1 and 0 < probs[i] <= 1
        if i < 4:
            assert ids[i] == (1 if s == MIXED[1] else by_logit[0])
        elif i < 8:
            want, _, _ = S.draw(x[i], *s, 1 - 2.0 ** -30)
            last = vocab - 2 if s == MIXED[1] else by_logit[6] if s[1] == 7 else None
            assert last is None or ids[i] in (last, want)


def test_infinities_and_nan(ctx, dev):
    rng = np.random.default_rng(4)
    vocab = 10000
    base = zipf(rng, 1, vocab)[0]
    rows = []
    for change in range(8):
        x = base.copy()
        if change == 0:
            x[rng.random(vocab) < 0.5] = -np.inf
        elif change == 1:
            x[rng.random(vocab) < 0.5] = np.nan
        elif change == 2:
            x[[700, 8000]] = np.inf
        elif change == 3:
            x[:] = -np.inf
        elif change == 4:
            x[:] = np.nan
        elif change == 5:
            x[:] = np.nan
            x[77], x[5000] = -np.inf, -np.inf
        elif change == 6:
            x[:] = -np.inf
            x[9999] = -1e30
        else:
            x[:5000] = np.where(rng.random(5000) < 0.5, 0.0, -0.0)
            x[5000:] = -3
        rows.append(x)
    sets = [MIXED[i] for i in (0, 1, 2, 6, 7, 11)]
    x = np.repeat(np.array(rows), len(sets), 0)
    Rows(dev, x, sets * 8, rng.random(len(x))).check(ctx)


def test_extreme_logits(ctx, dev):
    rng = np.random.default_rng(5)
    big = np.finfo(np.float32).max
    x = np.stack([rng.choice([big, -big, 0.0, 1.0], 3000), rng.standard_normal(3000) * 1e-42, rng.standard_normal(3000) * 1e30,
                  1e8 + 8.0 * rng.integers(0, 4, 3000)]).astype(np.float32)
    x = np.repeat(x, 5, 0)
    sets = [(1.0, 0, 1.0, 0.0), (0.5, 40, 0.9, 0.0), (1e30, 0, 0.9, 0.0), (1e-20, 3, 1.0, 0.0), (7.0, 0, 1.0, 0.2)] * 4
    Rows(dev, x, sets, rng.random(20)).check(ctx, 0.3)


def test_settings_that_are_refused(ctx, dev):
    """They end their own row alone."""
    rng = np.random.default_rng(6)
    nan, inf = float("nan"), float("inf")
    bad = [(nan, 0, 1.0, 0.0), (inf, 0, 1.0, 0.0), (1.0, -1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.5, 0.0), (1.0, 0, nan, 0.0),
           (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, -0.1), (1.0, 0, 1.0, nan), (0.0, -5, 1.0, 0.0)]
    sets = [s for b in bad for s in (b, MIXED[2])]
    x = zipf(rng, len(sets), 4000)
    r = Rows(dev, x, sets, rng.random(len(sets)))
    ids = r.check(ctx)
    assert (ids[::2] == -1).all() and (ids[1::2] >= 0).all()
    assert (r.read()[1][::2] == 0).all()


def test_against_the_sampler_of_one_row(ctx, dev):
    """The first draw of ihip_enqueue_sample's stream, whose number is the row's."""
    rng = np.random.default_rng(7)
    vocab = 151936
    x = zipf(rng, 8, vocab)
    sets = [MIXED[i] for i in (1, 2, 3, 4, 5, 6, 7, 14)]
    r = Rows(dev, x, sets, [splitmix(100 + i) for i in range(8)])
    ids = r.check(ctx)
    for i, (t, k, p, m) in enumerate(sets):
        s = H.Sampler(ctx, vocab, temperature=t, top_k=k, top_p=p, min_p=m, seed=100 + i)
        out = dev.out(4)
        s.enqueue(dev(x[i]), vocab, out.ptr)
        assert out.download(np.int32, 1)[0] == ids[i]
        s.close()


def test_without_probabilities_and_from_run_to_run(ctx, dev):
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((40, 60000)) * 2).astype(np.float32)
    r = Rows(dev, x, MIXED * 2, rng.random(40))
    r.enqueue(ctx)
    ids, probs = r.read()
    for _ in range(3):
        r.probs.upload(np.full(4 * 40 + 16, 0x5A, np.uint8))
        r.enqueue(ctx, probs=False)
        assert np.array_equal(r.read()[0], ids) and (r.probs.download(np.uint8, 160) == 0x5A).all()
        r.enqueue(ctx)
        assert np.array_equal(r.read()[1].view(np.uint32), probs.view(np.uint32))


def test_captured_and_replayed(ctx, dev):
    """Two graphs of one context over its workspace, replayed in turn as logits, settings and
    numbers change."""
    rng = np.random.default_rng(9)
    rs = [Rows(dev, zipf(rng, 5, 30000), MIXED[2:7], rng.random(5)), Rows(dev, zipf(rng, 33, 9000), (MIXED * 2)[:33], rng.random(33))]
    bufs = []
    for i, r in enumerate(rs):
        n, v = r.x.shape
        b = [dev.out(r.x.nbytes), dev.out(len(settings_array(r.settings))), dev.out(8 * n)]
        r.args = (b[0].ptr, n, v, 0, b[1].ptr, b[2].ptr)
        bufs.append(b)
        b[1].upload(settings_array(r.settings))  # (the kernels read settings when they run alone)
        H.check(H.lib().ihip_capture_begin(ctx.h))
        r.enqueue(ctx)
        H.check(H.lib().ihip_capture_end(ctx.h, 14 + i))
    for step in range(4):
        for i, r in enumerate(rs):
            n, v = r.x.shape
            r.x, r.u = zipf(rng, n, v), rng.random(n)
            r.settings = [MIXED[int(j)] for j in rng.integers(0, len(MIXED), n)]
            for b, a in zip(bufs[i], (r.x, settings_array(r.settings), r.u)):
                b.upload(a)
            H.check(H.lib().ihip_graph_launch(ctx.h, 14 + i))
        outs = [r.read() for r in rs]
        for r, (ids, probs) in zip(rs, outs):
            assert np.array_equal(r.check(ctx), ids) and np.array_equal(r.read()[1], probs)

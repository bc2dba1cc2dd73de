"""Draws of many rows on the host (no device): refused calls, the weights' whole numbers,
and the definition (sample_ref.py) against the oracle's TInferSampler."""
import numpy as np
import pytest

import infer_hip as H
import oracle_lib as O
import sample_ref as S
from test_paged import A, refused


def call(**kw):
    a = dict(ctx=None, x=A, rows=3, vocab=1000, stride=0, settings=2 * A, uniform=3 * A, ids=4 * A, probs=5 * A)
    a.update(kw)
    return H.lib().ihip_enqueue_sample_rows(*a.values())


def test_refused():
    for name in ("x", "settings", "uniform", "ids"):
        refused(lambda: call(**{name: 0}), -1, "missing array")
    for bad in (dict(rows=0), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(rows=-1)):
        refused(lambda: call(**bad), -1, "out of range")
    refused(lambda: call(stride=999), -1, "stride below")
    refused(lambda: call(stride=(1 << 36) + 1), -1, "2^36")
    for name in ("x", "ids", "probs"):
        refused(lambda: call(**{name: A + 2}), -1, "4 bytes")
    for name in ("settings", "uniform"):
        refused(lambda: call(**{name: A + 4}), -1, "8 bytes")
    refused(lambda: call(), -1, "no context")
    refused(lambda: call(probs=0), -1, "no context")


def test_overlaps_are_refused():
    # of 3 rows: 12 bytes of ids and of probs, logits 1000 floats every 1100, 40 bytes of settings, 8 of uniform
    for name in ("ids", "probs"):
        for at in (A - 8, A, A + 4 * 999, A + 4 * 1100 - 8, A + 4 * (2200 + 999), 2 * A - 8, 2 * A + 116, 3 * A - 8, 3 * A + 20):
            refused(lambda: call(stride=1100, **{name: at}), -1, "overlap")
        for at in (A - 12, A + 4 * 1000, A + 4 * 1100 - 12, A + 4 * (2200 + 1000), 2 * A - 12, 2 * A + 120, 3 * A - 12, 3 * A + 24):
            refused(lambda: call(stride=1100, **{name: at}), -1, "no context")
    for at in (4 * A - 8, 4 * A, 4 * A + 8):
        refused(lambda: call(probs=at), -1, "overlap")
    for at in (4 * A - 12, 4 * A + 12):
        refused(lambda: call(probs=at), -1, "no context")


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 1023, 1024, 1025, 1 << 21, (1 << 21) + 1, 1 << 22])
def test_weights_fit(vocab):
    """A vocabulary's weights (at most 1 each) add up below 2^62, and one is below 2^52."""
    bits = O.lib().orc_sample_weight_bits(vocab)
    assert vocab << bits < 1 << 62 and bits <= 51
    assert bits == 51 or vocab << bits + 2 > 1 << 62


def splitmix(seed):
    """The first number of a sampler's stream."""
    m = (1 << 64) - 1
    z = (seed + 0x9E3779B97F4A7C15) & m
    z = (z ^ z >> 30) * 0xBF58476D1CE4E5B9 & m
    z = (z ^ z >> 27) * 0x94D049BB133111EB & m
    return ((z ^ z >> 31) >> 11) / 2.0 ** 53


@pytest.mark.parametrize("vocab", [1, 2, 63, 500])
def test_definition_against_the_oracle(vocab):
    rng = np.random.default_rng(vocab)
    for seed in range(150):
        x = (rng.standard_normal(vocab) * rng.choice([0, 1, 6])).astype(np.float32)
        if seed % 3 == 0:
            x[rng.integers(0, vocab, 3)] = rng.choice([-np.inf, np.nan, 3.0, 3.0], 3)
        kw = dict(temperature=float(rng.choice([0, 0.5, 1, 3])), top_k=int(rng.choice([0, 0, 1, 5, 40])),
                  top_p=float(rng.choice([1, 1, 0.9, 0.3])), min_p=float(rng.choice([0, 0, 0.05, 0.5])))
        s = O.Sampler(seed=seed, **kw)
        got, _, margin = S.draw(x, u=splitmix(seed), **kw)
        want = s.next(x)
        s.close()
        assert got == want or margin < 1e-12, (seed, kw, got, want, margin)

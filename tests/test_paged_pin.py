"""The tolerance of paged_pin.py on the host: it sees one key left out or taken
twice at every border, and weights or queries of one part alone."""
import numpy as np
import pytest

import paged_pin as P

LENGTHS = [2, 17, 64, 129, 1000, 9000, 20000]


def case(n, hd, scale, seed=0):
    rng = np.random.default_rng(seed + n)
    k, v = rng.standard_normal((2, 1, n, 1, hd))
    q = rng.standard_normal((1, 2, hd))
    return q, k, v, np.zeros((1, 1), np.int32), [n], n, scale


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("hd,scale", [(64, 0.0), (128, 0.0), (128, 0.004), (512, 0.0)])
def test_one_key_is_seen(dtype, n, hd, scale):
    q, k, v, table, lengths, ps, scale = case(n, hd, scale)
    y, tol, held = P.attention(q, k, v, table, lengths, ps, dtype, scale=scale)
    for h in range(2):
        _, w, vv = held[0, h]
        for j in P.border_keys(n):
            assert min(P.least_change(y[0, h], w, vv, j)) > 2 * tol[0, h], (h, j)


@pytest.mark.parametrize("n", LENGTHS)
def test_half_the_bits_are_seen(n):
    """Weights, or queries, of one half (11 bits) instead of two."""
    q, k, v, table, lengths, ps, _ = case(n, 128, 0.0)
    y, tol, held = P.attention(q, k, v, table, lengths, ps, "f16")
    for h in range(2):
        _, w, vv = held[0, h]
        p = (w / w.max()).astype(np.float16).astype(np.float64)
        # (one key's weight, or two equal ones, may be a half)
        assert np.linalg.norm(p @ vv / (w / w.max()).sum() - y[0, h]) > 2 * tol[0, h]
    short, _, _ = P.attention(q.astype(np.float16).astype(np.float64), k, v, table, lengths, ps, "f16")
    assert (np.linalg.norm(short - y, axis=2) > 2 * tol).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_single_sums_pass(dtype):
    """numpy's own single sums over the keys, in one chain, stay within it."""
    for n in (64, 1000, 9000):
        q, k, v, table, lengths, ps, _ = case(n, 128, 0.0)
        q, k, v = (a.astype(np.float32) for a in (q, k, v))
        y, tol, _ = P.attention(*(a.astype(np.float64) for a in (q, k, v)), table, lengths, ps, dtype)
        for h in range(2):
            x = k[0, :, 0] @ (q[0, h] * np.float32(128 ** -0.5))
            p = np.exp(x - x.max())
            got = (p[:, None] * v[0, :, 0]).sum(0, dtype=np.float32) / p.sum(dtype=np.float32)
            assert np.linalg.norm(got - y[0, h]) < tol[0, h]

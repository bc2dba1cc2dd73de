"""Paged attention on the device within the tolerance of its own roundings
(paged_pin.py; test_paged_pin.py shows on the host that it sees one key left out
at every border of these lengths), and head sizes of 264 to 504."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_pin as P
import paged_ref as R
from test_gpu_paged import ctx, dev, pages_struct  # noqa: F401 (fixtures)
from test_paged_pin import LENGTHS

pytestmark = pytest.mark.gpu


def attend(ctx, dev, dtype, hd, heads, kvh, ps, lengths, window=0, sinks=False, scale=0.0, seed=0):
    rng = np.random.default_rng(seed + hd + heads)
    lengths = np.array(lengths, np.int32)
    have = -(-lengths // ps)
    pages, width, n = int(have.sum()) + 2, int(have.max()) + 1, len(lengths)
    order, table, at = rng.permutation(pages).astype(np.int32), np.full((n, width), -1, np.int32), 0
    for s in range(n):
        table[s, :have[s]] = order[at:at + have[s]]
        at += have[s]
    raw = [R.pack(rng.standard_normal((pages, ps, kvh, hd)), dtype) for _ in range(2)]
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    sk = rng.standard_normal(heads).astype(np.float32) if sinks else None
    y = dev.out(q.nbytes)
    pool = pages_struct(dev(raw[0]), dev(raw[1]), pages, ps, kvh, hd, dtype)
    H.check(H.lib().ihip_enqueue_paged_attention(
        ctx.h, dev(q), 0, C.byref(pool), dev(table), width, dev(lengths), y.ptr, n, heads, window,
        dev(sk) if sinks else 0, scale), "attention")
    got = y.download(np.float32, q.size).reshape(q.shape)
    want, tol, _ = P.attention(q.astype(np.float64), R.unpack(raw[0], dtype), R.unpack(raw[1], dtype), table, lengths,
                               ps, dtype, window, None if sk is None else sk.astype(np.float64), scale)
    off = np.linalg.norm(got - want, axis=2)
    assert (off <= tol).all(), (np.argwhere(off > tol)[:5].tolist(), (off / np.maximum(tol, 1e-300)).max())
    return (off / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd,heads,kvh,ps,most", [
    (64, 4, 2, 16, 20000), (128, 2, 1, 16, 20000), (128, 8, 2, 7, 9000), (96, 3, 3, 8, 1000), (256, 4, 2, 64, 9000),
    (512, 2, 1, 16, 9000), (128, 40, 2, 16, 1000), (200, 2, 1, 1, 1000)])
def test_attention_to_its_roundings(ctx, dev, dtype, hd, heads, kvh, ps, most):
    attend(ctx, dev, dtype, hd, heads, kvh, ps, [n for n in LENGTHS if n <= most])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("length", [9000, 20000])
def test_attention_of_one_long_sequence(ctx, dev, dtype, length):
    """Split over all blocks and joined in two levels; weights nearly equal, so that each key counts."""
    attend(ctx, dev, dtype, 128, 8, 1, 16, [length], scale=0.004)
    attend(ctx, dev, dtype, 128, 8, 1, 16, [length], sinks=True)
    attend(ctx, dev, dtype, 64, 2, 1, 100, [length], window=length - 77)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [264, 320, 384, 456, 504])
@pytest.mark.parametrize("heads,kvh,ps", [(2, 2, 16), (17, 1, 7)])
def test_attention_heads_beyond_256(ctx, dev, dtype, hd, heads, kvh, ps):
    """Two waves share a head's dimensions, and the second's end before 512."""
    attend(ctx, dev, dtype, hd, heads, kvh, ps, [1, 2, 15, 33, 64, 129, 1000])
    attend(ctx, dev, dtype, hd, heads, kvh, ps, [3000], sinks=True)
    attend(ctx, dev, dtype, hd, heads, kvh, ps, [77, 600, 5], window=40)

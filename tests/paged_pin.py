"""Attention over pages in 64 bits with a tolerance that follows the kernels'
own roundings: tight enough to see one key left out, or weights of half the bits.

The error of a head is taken over its dimensions together (its norm), where
independent roundings add as squares. With U half a step of single:

- a score, in base 2: each product of a query value off by U (the scaling), by 4 U more
  in halves, whose two parts hold 22 bits; the products' sum, at most hd roundings
  for each part, as squares, against the size of the partial sums, sqrt(sum q^2 k^2)
  (q with the scale in it, as below); U of the score for the scale, U of its distance
  to the maximum;
- a weight: ln 2 of its score's error, 2 U of the exponential, 4 U of two half parts;
- the sums over keys: one rounding a key and part of a lane's chain, then 84 of the waves'
  and the pieces' joins, as squares, against sqrt(sum w^2 v^2) or the result, the larger.
  A wave takes a quarter of a block's keys, and a launch has 256 blocks at least where
  there are tiles for them;
- the total, its division and the last rounding: 4 U of the result.

The tolerance is four times the root of the squares' sum."""
import numpy as np

import paged_ref as R

U = R.U
PARTS = {"f32": 1, "f16": 2, "bf16": 3}


def weights(q, k, keys, scale, sinks=None):
    """(x, w): the scaled scores of one head's keys in nature's base, their softmax."""
    x = k[keys[:, 0], keys[:, 1]] @ q * scale
    top = max(x.max(), sinks) if sinks is not None else x.max()
    e = np.exp(x - top)
    return x, e / (e.sum() + (np.exp(sinks - top) if sinks is not None else 0.0))


def attention(q, k, v, table, lengths, ps, dtype, window=0, sinks=None, scale=0.0):
    """(y [seqs, heads, hd], tol [seqs, heads], keys and weights of each head)"""
    seqs, heads, hd = q.shape
    kvh = k.shape[2]
    scale = scale or hd ** -0.5
    y, tol, held = np.zeros(q.shape), np.zeros((seqs, heads)), {}
    at = [np.array(R.keys_of(table[s], lengths[s], window, ps, k.shape[0])).reshape(-1, 2) for s in range(seqs)]
    tile = (64 if dtype == "f32" else 128) // (2 if hd > 256 else 1)
    tiles = sum(-(-len(a) // tile) for a in at) * kvh * -(-(heads // kvh) // 16)
    chain = -(-tiles // 256) * tile / 4
    half = 4 if dtype == "f16" else 0
    for s in range(seqs):
        if not len(at[s]):
            continue
        for h in range(heads):
            g = h // (heads // kvh)
            sink = None if sinks is None else float(sinks[h])
            x, w = weights(q[s, h], k[:, :, g], at[s], scale, sink)
            kk, vv = k[at[s][:, 0], at[s][:, 1], g], v[at[s][:, 0], at[s][:, 1], g]
            y[s, h] = w @ vv
            b = np.abs(x) / np.log(2)
            part = np.sqrt((kk * kk) @ (q[s, h] * q[s, h])) * scale / np.log(2)
            score = (1 + half + np.sqrt(PARTS[dtype] * hd)) * part + b + np.abs(x - x.max()) / np.log(2)
            off = np.log(2) * score + 2 + half
            e1 = (w * w * off * off) @ ((vv - y[s, h]) ** 2).sum(1)
            size = max(np.sqrt((w * w) @ (vv * vv).sum(1)), np.linalg.norm(y[s, h]))
            e2 = (chain * PARTS[dtype] + 84) * size * size
            e3 = (16 + chain + 84) * (y[s, h] ** 2).sum()
            tol[s, h] = 4 * U * np.sqrt(e1 + e2 + e3)
            held[s, h] = at[s], w, vv
    return y, tol, held


def border_keys(n):
    """Keys at the ends of steps, tiles and the whole."""
    at = {0, 1, n - 1, n - 2, n // 2}
    for step in (16, 32, 64, 128, 4096):
        for i in range(0, n + 1, step * max(1, n // (8 * step))):
            at |= {i - 1, i}
    return sorted(i for i in at if 0 <= i < n)


def least_change(y, w, vv, j):
    """The norm of what leaving key j out, or taking it twice, changes: the smaller."""
    d = np.linalg.norm(vv[j] - y)
    return w[j] * d / max(1 - w[j], 1e-300) if w[j] < 1 else np.inf, w[j] * d / (1 + w[j])

"""A draw by TInferSampler's definition in 64 bits (numpy), from a given random number."""
import numpy as np


def draw(x, temperature, top_k, top_p, min_p, u):
    """(id, probability among the kept, margin): margin is how near a comparison of sums or weights
    was to the other way, relative to the sums."""
    x = x.astype(np.float64)
    if not all(np.isfinite(v) for v in (temperature, top_p, min_p)) or top_k < 0 or not 0 < top_p <= 1 \
            or not 0 <= min_p < 1:
        return -1, 0.0, 1.0
    seen = np.where(np.isnan(x), -np.inf, x)
    # (the first index of the maximum, NaN skipped; 0 where all are NaN)
    best = int(np.flatnonzero(x == seen.max())[0]) if not np.isnan(x).all() else 0
    if temperature < 1e-30 or not np.isfinite(seen.max()):
        return best, 1.0, 1.0
    w = np.where(np.isfinite(x), np.exp((np.where(np.isfinite(x), x, -np.inf) - seen.max()) / temperature), 0.0)
    margin = 1.0
    if top_k == 0 and top_p >= 1 and min_p == 0:
        at, p = np.arange(len(x)), w
    else:
        at = np.lexsort((np.arange(len(x)), -seen))
        at = at[np.isfinite(x[at])]
        if 0 < top_k < len(at):
            at = at[x[at] >= x[at[top_k - 1]]]
        if top_p < 1:
            run = np.cumsum(w[at])
            mass = run[-1] if top_k > 0 else w.sum()
            before = np.concatenate([[0.0], run[:-1]])
            keep = before < top_p * mass
            keep[0] = True
            margin = min(margin, np.abs(run - top_p * mass).min() / mass)
            at = at[keep]
        if min_p > 0:
            keep = w[at] >= min_p
            keep[0] = True
            margin = min(margin, np.abs(w[at] - min_p).min())
            at = at[keep]
        p = w[at]
    run = np.cumsum(p)
    hit = np.flatnonzero((u * run[-1] < run) & (p > 0))
    i = int(hit[0]) if len(hit) else (int(np.argmax(at == best)))
    margin = min(margin, np.abs(run - u * run[-1]).min() / run[-1])
    return int(at[i]), p[i] / run[-1], margin

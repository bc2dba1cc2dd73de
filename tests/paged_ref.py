"""The paged operators in 64 bits, from their definitions (numpy, no device): the
oracle of test_paged.py, test_gpu_paged.py and test_gpu_logprobs.py."""
import numpy as np

U = 2.0 ** -24  # half a step of single
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def bf16_bits(a):
    """Single values rounded to bf16 (nearest, ties to even), as uint16."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def pack(a, dtype):
    return a.astype(np.float32) if dtype == "f32" else a.astype(np.float16) if dtype == "f16" \
        else bf16_bits(a)


def unpack(raw, dtype):
    """The values of a cache's elements, in 64 bits."""
    if dtype == "bf16":
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.astype(np.float64)


def slots(past, count, table, page_size, ring, ends, rows):
    """The plan of a step, sequence after sequence."""
    table, ring, free = table.copy(), ring.copy(), ring.copy()
    pages, width = len(ring), table.shape[1]
    first, last = (int(e) for e in ends)
    avail = min(last - first, pages) if first >= 0 and last > first else 0
    wanted = put = failed = taken = back = 0
    offsets, lengths, positions, out = [0], [], [], []
    for s in range(len(past)):
        a, n = int(past[s]), 1 if count is None else int(count[s])
        if a < 0 or n < 0:
            lengths.append(-1)
            offsets.append(offsets[-1])
            if a >= 0:
                have = min(-(-a // page_size), width)
                put += have
                if put <= pages - avail:
                    for p in table[s, :have]:
                        ring[(last + back) % pages] = p
                        back += 1
            continue
        have = -(-a // page_size)
        offsets.append(offsets[-1] + n)
        ok = a + n <= width * page_size and offsets[-1] <= rows
        if ok:
            need = -(-(a + n) // page_size) - have
            wanted += need
            ok = need == 0 or wanted <= avail
        if ok:
            for j in range(need):
                table[s, have + j] = free[(first + taken) % pages]
                taken += 1
        failed += not ok
        lengths.append(a + n if ok else a)
        for p in range(a, a + n):
            e = int(table[s, p // page_size]) if ok else -1
            positions.append(p)
            out.append(e * page_size + p % page_size if 0 <= e < pages else -1)
    pad = [-1] * max(0, rows - len(positions))

    def i32(a):
        return np.array(a, np.int32)

    return dict(table=table, ring=ring, ends=np.array([first + taken, last + back], np.int64),
                offsets=i32(offsets), lengths=i32(lengths), positions=i32((positions + pad)[:rows]),
                slots=i32((out + pad)[:rows]), failed=i32([failed]))


def rope(x, w, eps, freq, dims, interleaved, scale, positions):
    """x [rows, heads, hd]: the norm (w or None), then the rotation (freq or None)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    if freq is None:
        return x
    ang = freq.astype(np.float64)[None] * positions.astype(np.float64)[:, None]
    c, s = (f(ang)[:, None] * scale for f in (np.cos, np.sin))
    y = x.copy()
    i0, i1 = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else \
        (slice(0, dims // 2), slice(dims // 2, dims))
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def keys_of(table, length, window, page_size, pages):
    """(page, token) of the keys that a sequence's new token sees."""
    n = min(max(int(length), 0), len(table) * page_size)
    out = []
    for j in range(max(0, n - window) if window else 0, n):
        p = int(table[j // page_size])
        if 0 <= p < pages:
            out.append((p, j % page_size))
    return out


def attention(q, k, v, table, lengths, page_size, window=0, sinks=None, scale=0.0):
    """q [seqs, heads, hd], k and v [pages, page_size, kv_heads, hd] in 64 bits. Returns (y, tol):
    tol bounds what sums in single may be off by, in any order and with a running maximum. A
    score: hd products and sums, each off by U of the magnitudes' sum. A weight: twice its
    score's error (its own, the maximum's) and the exponential's, 8 U. The sums over n keys:
    2 n + 32 roundings of magnitudes (n additions, as many rescales, the joins)."""
    seqs, heads, hd = q.shape
    group = heads // k.shape[2]
    scale = scale if scale > 0 else hd ** -0.5
    y, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(seqs):
        at = keys_of(table[s], lengths[s], window, page_size, k.shape[0])
        if lengths[s] < 0 or not at:
            continue
        pg, tk = (np.array(i) for i in zip(*at))
        for h in range(heads):
            kk, vv = k[pg, tk, h // group], v[pg, tk, h // group]
            x = kk @ q[s, h] * scale
            off = (hd + 8) * U * (np.abs(kk) @ np.abs(q[s, h])) * scale
            top = max(x.max(), sinks[h]) if sinks is not None else x.max()
            e = np.exp(x - top)
            den = e.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0)
            y[s, h] = e @ vv / den
            rel = 2 * off.max() + (np.abs(x - top) * e).sum() / den * 4 * U + (2 * len(x) + 40) * U
            tol[s, h] = rel * (e @ np.abs(vv) / den + np.abs(y[s, h])) + 1e-37
    return y, tol


def order(row):
    """The ids of a row's logits, the largest first, the lowest id on a tie, NaN last."""
    key = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    return np.lexsort((np.arange(len(row)), -key, np.isnan(row)))


def logprobs(x, ids, k):
    """(logprobs, entropy, top_ids, top_logprobs) and tolerances of the three floats. In single a
    difference to the maximum is off by U of itself, an exponential by 4 U, their sums (in
    parts of 8 in single, then double) by 8 U, and the result is rounded."""
    rows, vocab = x.shape
    lp, ent = np.full(rows, np.nan), np.full(rows, np.nan)
    top_ids, top = np.full((rows, k), -1, np.int32), np.full((rows, k), -np.inf)
    tol_lp, tol_ent, tol_top = np.zeros(rows), np.zeros(rows), np.zeros((rows, k))
    for r in range(rows):
        d = x[r].astype(np.float64)
        n = min(k, vocab)
        top_ids[r, :n] = order(x[r])[:n]
        if np.isnan(d).any() or (d == np.inf).any():
            top[r, :n] = np.nan
            continue
        if (d == -np.inf).all():
            l, ent[r], mean = d, 0.0, 0.0
        else:
            d = d - d.max()
            e = np.exp(d)
            tot = e.sum()
            l = d - np.log(tot)
            fin = e > 0
            mean = (e[fin] * -d[fin]).sum() / tot
            ent[r] = np.log(tot) + mean
            sq = (e[fin] * d[fin] ** 2).sum() / tot
            tol_ent[r] = U * (2 * ent[r] + 20 * mean + 2 * sq + 16 + mean * mean)
        base = 2 * mean + 16
        if ids is not None and 0 <= ids[r] < vocab:
            lp[r] = l[ids[r]]
        tol = U * (4 * np.abs(np.where(np.isfinite(l), l, 0)) + base)
        if ids is not None and 0 <= ids[r] < vocab:
            tol_lp[r] = tol[ids[r]]
        top[r, :n], tol_top[r, :n] = l[top_ids[r, :n]], tol[top_ids[r, :n]]
    return lp, ent, top_ids, top, tol_lp, tol_ent, tol_top

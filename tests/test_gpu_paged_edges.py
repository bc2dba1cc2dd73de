"""The paged operators on the device at the edges of what a call may hold,
against paged_ref.py's definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_ref as R
from test_gpu_paged import assert_close, batch, ctx, dev, pages_struct, run_slots  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------- attention
class Batch:
    """Keys, values, tables and queries of a batch, by default of full pages of its own each."""

    def __init__(self, rng, dtype, hd, heads, kvh, ps, lengths, width=None):
        self.dtype, self.hd, self.heads, self.kvh, self.ps = dtype, hd, heads, kvh, ps
        self.lengths = np.array(lengths, np.int32)
        n = len(lengths)
        self.width = width or max(1, int((-(-self.lengths.clip(0) // ps)).max()))
        self.pages = n * self.width
        self.table = rng.permutation(self.pages).reshape(n, self.width).astype(np.int32)
        self.k, self.v = (rng.standard_normal((self.pages, ps, kvh, hd)) for _ in range(2))
        self.q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        self.sinks, self.window, self.scale = None, 0, 0.0

    def upload(self, dev):
        self.raw = [R.pack(a, self.dtype) for a in (self.k, self.v)]
        self.pool = pages_struct(dev(self.raw[0]), dev(self.raw[1]), self.pages, self.ps, self.kvh, self.hd, self.dtype)
        self.dq, self.dt, self.dl = dev(self.q), dev(self.table), dev(self.lengths)
        self.ds = dev(self.sinks) if self.sinks is not None else 0
        self.y = dev.out(self.q.nbytes)

    def enqueue(self, ctx):
        H.check(H.lib().ihip_enqueue_paged_attention(
            ctx.h, self.dq, 0, C.byref(self.pool), self.dt, self.width, self.dl, self.y.ptr, len(self.lengths),
            self.heads, self.window, self.ds, self.scale), "attention")

    def read(self):
        return self.y.download(np.float32, self.q.size).reshape(self.q.shape)

    def want(self):
        with np.errstate(invalid="ignore", over="ignore"):
            return R.attention(self.q.astype(np.float64), R.unpack(self.raw[0], self.dtype),
                               R.unpack(self.raw[1], self.dtype), self.table, self.lengths, self.ps, self.window,
                               self.sinks, self.scale)

    def run(self, ctx, dev):
        self.upload(dev)
        self.enqueue(ctx)
        return self.read()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 3, 5, 9])
def test_attention_by_rows_without_offsets(ctx, dev, dtype, rows):
    """Row s of sequence s where q and y have one; the other sequences are passed over."""
    rng = np.random.default_rng(rows)
    b = Batch(rng, dtype, 64, 4, 2, 16, [40, 0, 33, 1, 70])
    b.upload(dev)
    H.check(H.lib().ihip_enqueue_paged_attention_at(
        ctx.h, b.dq, 0, C.byref(b.pool), b.dt, b.width, b.dl, 0, rows, b.y.ptr, 5, b.heads, 0, 0, 0.0), "attention")
    got, (want, tol) = b.read(), b.want()
    assert_close(got[:rows], want[:rows], tol[:rows])
    assert (got[rows:].view(np.uint8) == 0x5A).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("off", [-np.inf, np.finfo(np.float32).min])
def test_attention_sinks_switched_off(ctx, dev, dtype, off):
    """A sink of -infinity, or one that its scaling makes so, has no weight: sequences whose keys are
    none, all outside the pool, or all of score -infinity (in one piece, and split over the length)
    give zeros, the others what they give without a sink."""
    rng = np.random.default_rng(11)
    b = Batch(rng, dtype, 128, 8, 2, 16, [50, 0, 64, 9000, 9000, 200])
    b.table[0, :] = -1
    b.table[4, :] = b.pages + 3
    b.q = np.abs(b.q)
    for s in (2, 3):  # scores of -infinity, whatever the query
        b.k[b.table[s], :, :, 5] = -np.inf
    b.sinks = rng.standard_normal(8).astype(np.float32)
    b.sinks[[0, 3, 5]] = off
    got, (want, tol) = b.run(ctx, dev), (None, None)
    assert (got[:5] == 0).all(), np.isnan(got[:5]).sum((1, 2))
    want, tol = b.want()
    assert_close(got[5], want[5], tol[5])
    b.sinks[1], b.sinks[4] = np.nan, np.inf
    got = b.run(ctx, dev)
    assert np.isnan(got[5, 1]).all() and (got[5, 4] == 0).all()
    others = [0, 2, 3, 5, 6, 7]
    assert_close(got[5][others], want[5][others], tol[5][others])


# ---------------------------------------------------------------------- plan
def plan_with_holes(past, count, table, page_size, ring, ends, rows):
    """The plan in which an ended sequence holds the pages of the pool that its table has, and no
    others; the table itself is left as it is."""
    t, held = table.copy(), past.copy()
    ended = np.flatnonzero((past >= 0) & (count < 0))
    for s in ended:
        have = min(-(-int(past[s]) // page_size), t.shape[1])
        own = t[s, :have]
        own = own[(own >= 0) & (own < len(ring))]
        t[s, :len(own)], held[s] = own, len(own) * page_size
    want = R.slots(held, count, t, page_size, ring, ends, rows)
    want["table"][ended] = table[ended]
    return want


@pytest.mark.parametrize("n,page_size,most,new,spare,rows", [
    (1, 16, 900, 1, 4, 1), (3, 1, 300, 3, 20, 16), (64, 16, 300, 1, 64, 64), (200, 24, 500, 40, 500, 9000),
    (257, 4, 700, 9, 300, 4097), (1000, 3, 20, 9, 4000, 3000), (4096, 2, 30, 2, 2000, 12000)])
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
def test_slots_ended_tables_with_holes(ctx, dev, n, page_size, most, new, spare, rows, share):
    """An ended sequence's entries outside the pool (a window's pages, released before) do not come
    into the ring, and those behind them do, in order."""
    rng = np.random.default_rng(n + int(100 * share))
    past, count, table, ring, ends = batch(rng, n, page_size, most, new, spare, ended=0.4)
    if n == 1:
        past[:], count[:] = most, -1
        table[:, :-(-most // page_size)] = np.arange(-(-most // page_size)) % len(ring)
    ended = np.flatnonzero(count < 0)
    hole = rng.random((len(ended), table.shape[1])) < share
    bad = rng.choice(np.array([-1, -2 ** 31, len(ring), 2 ** 31 - 1], np.int32), hole.shape)
    table[ended] = np.where(hole, bad, table[ended])
    want = plan_with_holes(past, count, table, page_size, ring, ends, rows)
    got = run_slots(ctx, dev, past, count, table, page_size, ring, ends, rows)
    for k in want:
        if k != "ring":
            assert np.array_equal(got[k], want[k]), k
    # the free pages (what the ring holds outside its ends is nothing)
    at = np.arange(*want["ends"]) % len(ring)
    assert np.array_equal(got["ring"][at], want["ring"][at])
    assert len(set(at.tolist())) == len(at)


def test_slots_shared_pages_ended(ctx, dev):
    """Two sequences over a common prompt: the one that ends first has the shared entries taken out of
    its table, and only its own pages are free afterwards; then all pages are given out once."""
    ps, width, pages = 4, 8, 12
    table = np.full((3, width), -1, np.int32)
    table[0, :4], table[1, :4] = (3, 7, 1, 9), (3, 7, 0, 4)
    ring = np.array([2, 5, 6, 8, 10, 11, -7, -7, -7, -7, -7, -7], np.int32)
    past, ends = np.array([16, 16, 0], np.int32), np.array([0, 6], np.int64)
    table[1, :2] = -1
    got = run_slots(ctx, dev, past, np.array([1, -1, 1], np.int32), table, ps, ring, ends, 2)
    assert got["ends"].tolist() == [2, 8] and got["ring"][6:8].tolist() == [0, 4]
    assert got["table"][0, :5].tolist() == [3, 7, 1, 9, 2] and got["failed"][0] == 0
    past = got["lengths"].copy()
    past[1] = 0
    got = run_slots(ctx, dev, past, np.array([0, 24, 0], np.int32), got["table"], ps, got["ring"], got["ends"], 30)
    held = np.concatenate([got["table"][0, :5], got["table"][1, :6], got["table"][2, :1]])
    assert sorted(held.tolist()) == list(range(pages)) and got["failed"][0] == 0
    assert (got["slots"][:24] >= 0).all() and got["ends"].tolist() == [8, 8]
    # none is left
    got = run_slots(ctx, dev, got["lengths"], np.array([0, 1, 0], np.int32), got["table"], ps, got["ring"], got["ends"], 3)
    assert got["failed"][0] == 1 and got["slots"][0] == -1


# ------------------------------------------------------------------ together
def test_failed_sequence_in_a_step(ctx, dev):
    """A sequence that finds no page has its row in the step all the same: nothing is stored for it, and
    the attention answers the row from the keys that the sequence had; the others go on."""
    rng = np.random.default_rng(41)
    heads, kvh, hd, ps, width, n, pages = 4, 2, 64, 4, 6, 3, 5
    table = np.full((n, width), -1, np.int32)
    table[0, :2], table[1, :2] = (4, 0), (2, 1)
    ring, ends = np.array([3, -7, -7, -7, -7], np.int32), np.array([0, 1], np.int64)
    past, count = np.array([7, 8, 4], np.int32), np.array([1, 1, 1], np.int32)
    table[2, 0] = 1  # (its page is shared: it has one key more to come, and no page left for it)
    got = run_slots(ctx, dev, past, count, table, ps, ring, ends, n)
    assert got["failed"][0] == 1 and got["lengths"].tolist() == [8, 9, 4]
    assert got["offsets"].tolist() == [0, 1, 2, 3] and got["positions"].tolist() == [7, 8, 4]
    assert got["slots"].tolist() == [3, 3 * ps, -1]
    k, v = (rng.standard_normal((pages, ps, kvh, hd)).astype(np.float32) for _ in range(2))
    x = rng.standard_normal((n, heads + 2 * kvh, hd)).astype(np.float32)
    dk, dv = dev.out(k.nbytes), dev.out(v.nbytes)
    dk.upload(k), dv.upload(v)
    pool = pages_struct(dk.ptr, dv.ptr, pages, ps, kvh, hd, "f32")
    dx, y, row = dev(x), dev.out(n * heads * hd * 4), (heads + 2 * kvh) * hd
    H.check(H.lib().ihip_enqueue_paged_qkrope(
        ctx.h, dx, row, dx + 4 * heads * hd, row, dx + 4 * (heads + kvh) * hd, row, n, heads, 0, 0, 0.0, None,
        dev(got["positions"]), dev(got["slots"]), C.byref(pool), 0))
    H.check(H.lib().ihip_enqueue_paged_attention_at(
        ctx.h, dx, row, C.byref(pool), dev(got["table"]), width, dev(got["lengths"]), dev(got["offsets"]), n, y.ptr, n,
        heads, 0, 0, 0.0))
    for i, cache in enumerate((k, v)):
        at = cache.reshape(pages * ps, kvh, hd)
        at[[3, 3 * ps]] = x[:2, heads + i * kvh:heads + (i + 1) * kvh]
    assert np.array_equal(dk.download(np.float32, k.size), k.ravel())
    assert np.array_equal(dv.download(np.float32, v.size), v.ravel())
    want, tol = R.attention(x[:, :heads].astype(np.float64), k.astype(np.float64), v.astype(np.float64), got["table"],
                            got["lengths"], ps)
    assert_close(y.download(np.float32, want.size).reshape(want.shape), want, tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("sinks", [False, True])
def test_attention_scores_of_minus_infinity(ctx, dev, dtype, sinks):
    """A key of score -infinity has weight 0 and the others theirs; the KV head that does not see the
    infinity has its keys all."""
    rng = np.random.default_rng(6)
    b = Batch(rng, dtype, 128, 8, 2, 1, [48, 200, 5, 3000])
    b.q = np.abs(b.q)
    if sinks:
        b.sinks = rng.standard_normal(8).astype(np.float32)
    b.upload(dev)
    plain, _ = b.want()
    hidden = [(s, j) for s, n in enumerate(b.lengths) for j in (0, 3, n // 2, n - 1)]
    for s, j in hidden:
        b.k[b.table[s, j], 0, 1, 7] = -np.inf
    got = b.run(ctx, dev)
    b.k[~np.isfinite(b.k)] = 0  # (as a key that is not there)
    b.raw[0], table = R.pack(b.k, dtype), b.table.copy()
    want, tol = b.want()
    assert_close(got[:, :4], want[:, :4], tol[:, :4])
    for s, j in hidden:
        b.table[s, j] = -1
    want, tol = b.want()
    b.table = table
    assert_close(got[:, 4:], want[:, 4:], tol[:, 4:])
    assert np.abs(got[2, 4:] - plain[2, 4:]).max() > 1e-2  # (4 of 5 keys fewer)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_lengths_beyond_the_table(ctx, dev, dtype):
    """A length that the table does not hold is cut to it, every page of which is there; a window is the
    last keys of those."""
    rng = np.random.default_rng(13)
    for window in (0, 20):
        b = Batch(rng, dtype, 128, 8, 2, 16, [2 ** 31 - 1, 80, 81, 79, 5000], width=5)
        b.window = window
        got = b.run(ctx, dev)
        want, tol = b.want()
        assert_close(got, want, tol)
        b.lengths = np.array([80, 80, 80, 79, 80], np.int32)
        again, _ = b.want()
        assert np.array_equal(want, again)


def test_two_contexts_at_once(ctx):
    """Calls of two contexts on their own streams, all enqueued before the first is read."""
    rng = np.random.default_rng(32)
    with H.Context(0) as other:
        class Dev:
            def __init__(self, c):
                self.c = c

            def __call__(self, a):
                return self.c.array(a).ptr

            def out(self, nbytes, fill=0x5A):
                return self.c.array(np.full(nbytes, fill, np.uint8))

        calls = []
        for i in range(4):
            for c in (ctx, other):
                b = Batch(rng, ("f16", "bf16")[i % 2], 128, 16, 2, 16, [1500 + 100 * i, 3, 700, 4000])
                b.upload(Dev(c))
                calls.append((c, b))
        for _ in range(3):
            for c, b in calls:
                b.enqueue(c)
        for c, b in calls:
            want, tol = b.want()
            assert_close(b.read(), want, tol)
        ctx.sync()


@pytest.mark.parametrize("rows", [40, 9000])
def test_slots_windows_released(ctx, dev, rows):
    """Sequences of which only the last pages are left in a small pool, the others released by the host:
    the entries of those that end pass the pool's size many times, their pages come back all."""
    rng = np.random.default_rng(rows)
    n, ps, width, keep = 20, 16, 700, 6
    pages = n * keep + 30
    past = rng.integers(9000, 11000, n).astype(np.int32)
    have = -(-past // ps)
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    for s in range(n):
        table[s, have[s] - keep:have[s]] = order[s * keep:(s + 1) * keep]
    ring = np.full(pages, -7, np.int32)
    ring[:30] = order[n * keep:]
    count = np.where(np.arange(n) % 3 == 0, -1, 1).astype(np.int32)
    if rows > 4096:
        count[1] = 100
    ends = np.array([0, 30], np.int64)
    want = plan_with_holes(past, count, table, ps, ring, ends, rows)
    got = run_slots(ctx, dev, past, count, table, ps, ring, ends, rows)
    assert want["ends"][1] == 30 + keep * 7
    for k in want:
        if k != "ring":
            assert np.array_equal(got[k], want[k]), k
    at = np.arange(*want["ends"]) % pages
    assert np.array_equal(got["ring"][at], want["ring"][at])
    used = got["table"][count >= 0]
    used = used[(used >= 0) & (used < pages)]
    assert sorted(np.concatenate([used, got["ring"][at]]).tolist()) == list(range(pages))


@pytest.mark.parametrize("rows", [64, 5000])
def test_slots_with_holes_captured(ctx, dev, rows):
    """One graph over several batches, with holes and without, in place: what the blocks leave for each
    other is as it was before."""
    rng = np.random.default_rng(rows)
    n, ps, width = 40, 4, 40
    shape = dict(past=n, count=n, table=n * width, ring=2000, ends=2)
    b = {k: dev.out(m * (8 if k == "ends" else 4)) for k, m in shape.items()}
    o, q, s, f = dev.out(4 * n + 4), dev.out(4 * rows), dev.out(4 * rows), dev.out(4)

    def step():
        H.check(H.lib().ihip_enqueue_paged_slots(
            ctx.h, b["past"].ptr, b["count"].ptr, n, b["table"].ptr, width, ps, b["ring"].ptr, 2000, b["ends"].ptr,
            b["ends"].ptr, o.ptr, b["past"].ptr, q.ptr, s.ptr, rows, f.ptr))

    H.check(H.lib().ihip_capture_begin(ctx.h))
    step()
    H.check(H.lib().ihip_capture_end(ctx.h, 13))
    for i in range(8):
        past, count = rng.integers(0, 120, n).astype(np.int32), rng.integers(-1, 20, n).astype(np.int32)
        order = rng.permutation(2000).astype(np.int32)
        table = order[:n * width].reshape(n, width).copy()
        have = -(-past // ps)
        table[np.arange(width) >= have[:, None]] = -1
        if i % 3:
            table[(rng.random(table.shape) < 0.3) & (count < 0)[:, None]] = 2 ** 31 - 1
        ring, ends = np.full(2000, -7, np.int32), np.array([1900 + 2000 * i, 2300 + 2000 * i], np.int64)
        ring[np.arange(*ends) % 2000] = order[n * width:]
        for k, a in dict(past=past, count=count, table=table, ring=ring, ends=ends).items():
            b[k].upload(a)
        want = plan_with_holes(past, count, table, ps, ring, ends, rows)
        H.check(H.lib().ihip_graph_launch(ctx.h, 13))
        for k, d, dt in (("table", b["table"], np.int32), ("ends", b["ends"], np.int64), ("lengths", b["past"], np.int32),
                         ("slots", s, np.int32), ("positions", q, np.int32), ("offsets", o, np.int32),
                         ("failed", f, np.int32)):
            assert np.array_equal(d.download(dt, want[k].size), want[k].ravel()), (i, k)
        at = np.arange(*want["ends"]) % 2000
        assert np.array_equal(b["ring"].download(np.int32, 2000)[at], want["ring"][at]), i
        if i % 2:  # an eager call between the replays
            run_slots(ctx, dev, past, count, table, ps, ring, ends, rows)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_in_place(ctx, dev, dtype):
    """y in q's own rows: whole pieces, split ones, rows without a key, and one with an infinity."""
    rng = np.random.default_rng(23)
    b = Batch(rng, dtype, 128, 40, 2, 16, [50, 0, 9000, 1, -1, 70])
    b.k[b.table[5, 0], 3, 0, 9] = np.inf
    apart = b.run(ctx, dev)
    y = dev.out(b.q.nbytes)
    y.upload(b.q)
    b.dq, b.y = y.ptr, y
    b.enqueue(ctx)
    got = b.read()
    # bit for bit, NaN among them, and the place that is passed over holds its query
    assert np.array_equal(got[[0, 1, 2, 3, 5]].view(np.uint32), apart[[0, 1, 2, 3, 5]].view(np.uint32))
    assert np.array_equal(got[4], b.q[4])
    nan = np.zeros(40, bool)
    nan[:20] = b.q[5, :20, 9] > 0  # (a score of infinity; of -infinity the key has no weight)
    assert np.isnan(got[5][nan]).all() and np.isfinite(got[5][~nan]).all() and 0 < nan.sum() < 20

"""The paged operators on the device against their definitions in 64 bits
(paged_ref.py): the step plan, q/k/v into the pages, attention over them, and a
run of them together, captured and replayed."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_ref as R

pytestmark = pytest.mark.gpu
CODE = {"f32": H.F32, "f16": H.F16, "bf16": H.BF16}
U = R.U


@pytest.fixture(scope="module")
def ctx():
    c = H.Context(0)
    yield c
    c.close()


@pytest.fixture()
def dev(ctx):
    """Uploads that are freed with the test."""
    bufs = []

    class Dev:
        def __call__(self, a):
            bufs.append(ctx.array(a))
            return bufs[-1].ptr

        def out(self, nbytes, fill=0x5A):
            b = ctx.alloc(nbytes)
            b.upload(np.full(nbytes, fill, np.uint8))
            bufs.append(b)
            return b

    yield Dev()
    ctx.sync()
    for b in bufs:
        b.free()


# --------------------------------------------------------------------- slots
def run_slots(ctx, dev, past, count, table, page_size, ring, ends, rows, in_place=False):
    n, width = table.shape
    past, t, r, e = (np.ascontiguousarray(x) for x in (past, table, ring, ends))
    dp, dt, dr, de = (dev.out(x.nbytes) for x in (past, t, r, e))
    for b, x in ((dp, past), (dt, t), (dr, r), (de, e)):
        b.upload(x)
    do, dl = dev.out((n + 1) * 4), dp if in_place else dev.out(n * 4)
    dx = de if in_place else dev.out(16)
    ds, dq, df = dev.out(rows * 4 + 16), dev.out(rows * 4 + 16), dev.out(4)
    dc = dev(count) if count is not None else 0
    H.check(H.lib().ihip_enqueue_paged_slots(
        ctx.h, dp.ptr, dc, n, dt.ptr, width, page_size, dr.ptr, len(ring), de.ptr, dx.ptr, do.ptr,
        dl.ptr, dq.ptr, ds.ptr, rows, df.ptr), "slots")
    got = dict(table=dt.download(np.int32, t.size).reshape(t.shape),
               ring=dr.download(np.int32, len(ring)), ends=dx.download(np.int64, 2),
               offsets=do.download(np.int32, n + 1), lengths=dl.download(np.int32, n),
               positions=dq.download(np.int32, rows), slots=ds.download(np.int32, rows),
               failed=df.download(np.int32, 1))
    # nothing behind the rows is written
    for b in (ds, dq):
        assert (b.download(np.uint8, rows * 4 + 16)[rows * 4:] == 0x5A).all()
    return got


def batch(rng, n, page_size, most, new, spare, empty=0.1, ended=0.1):
    past = rng.integers(0, most + 1, n).astype(np.int32)
    past[rng.random(n) < empty] = -1
    count = rng.integers(0, new + 1, n).astype(np.int32)
    count[rng.random(n) < ended] = -1
    width = -(-(most + new) // page_size)
    have = -(-np.maximum(past, 0) // page_size)
    pages = int(have.sum()) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for s in range(n):
        table[s, :have[s]] = order[at:at + have[s]]
        at += have[s]
    # the free pages anywhere in the ring, past its end among them
    first = int(rng.integers(0, 3 * pages))
    ring = np.full(pages, -7, np.int32)
    for i in range(spare):
        ring[(first + i) % pages] = order[at + i]
    return past, count, table, ring, np.array([first, first + spare], np.int64)


@pytest.mark.parametrize("n,page_size,most,new,spare,rows", [
    (1, 16, 40, 1, 4, 1), (1, 1, 0, 1, 3, 5), (3, 7, 50, 3, 20, 16), (64, 16, 300, 1, 64, 64),
    (65, 16, 300, 2, 5, 130), (200, 24, 500, 40, 500, 9000), (257, 100, 64, 90, 100, 4096),
    (257, 100, 64, 90, 300, 4097), (1000, 3, 20, 9, 4000, 3000), (4096, 8, 30, 2, 2000, 12000),
    (4096, 16, 30, 1, 5000, 4096)])
@pytest.mark.parametrize("in_place", [False, True])
def test_slots(ctx, dev, n, page_size, most, new, spare, rows, in_place):
    rng = np.random.default_rng(n * 31 + page_size)
    past, count, table, ring, ends = batch(rng, n, page_size, most, new, spare)
    want = R.slots(past, count, table, page_size, ring, ends, rows)
    got = run_slots(ctx, dev, past, count, table, page_size, ring, ends, rows, in_place)
    for k in want:
        assert np.array_equal(got[k], want[k]), k


def test_slots_default_count_and_edges(ctx, dev):
    rng = np.random.default_rng(9)
    past, _, table, ring, ends = batch(rng, 5, 4, 30, 1, 9)
    want = R.slots(past, None, table, 4, ring, ends, 5)
    got = run_slots(ctx, dev, past, None, table, 4, ring, ends, 5)
    for k in want:
        assert np.array_equal(got[k], want[k]), k
    # lengths beyond every table, huge counts, ends that count nothing: no place, no page
    big = 2 ** 31 - 1
    past = np.array([big, 3, big, 0, 7], np.int32)
    count = np.array([big, big, -1, 2, 1], np.int32)
    for e in ((5, 5), (9, 2), (-3, 4)):
        e = np.array(e, np.int64)
        got = run_slots(ctx, dev, past, count, table, 4, ring, e, 6)
        assert got["failed"][0] >= 2 and (got["ends"][0] == e[0])
        assert got["lengths"].tolist()[:3] == [big, 3, -1]
        assert (got["slots"] == -1).all()


def test_slots_ring_turned_often(ctx, dev):
    """Ends beyond 32 bits."""
    rng = np.random.default_rng(10)
    past, count, table, ring, ends = batch(rng, 40, 4, 30, 3, 50)
    for turns in (2 ** 33, 2 ** 45 + 7):
        e = ends + turns * len(ring)
        want = R.slots(past, count, table, 4, ring, e, 120)
        got = run_slots(ctx, dev, past, count, table, 4, ring, e, 120)
        for k in want:
            assert np.array_equal(got[k], want[k]), k


def test_slots_captured(ctx, dev):
    """Decode steps replayed from one graph: lengths, pages and the ring go on from replay to
    replay, in place."""
    rng = np.random.default_rng(4)
    past, _, table, ring, ends = batch(rng, 9, 4, 10, 20, 60, ended=0)
    table = np.ascontiguousarray(np.pad(table, ((0, 0), (0, 8)), constant_values=-1))
    n, width = table.shape
    bufs = {}
    for k, a in dict(past=past, table=table, ring=ring, ends=ends).items():
        bufs[k] = dev.out(a.nbytes)
        bufs[k].upload(a)
    o, q, s, f = dev.out(4 * n + 4), dev.out(4 * n), dev.out(4 * n), dev.out(4)

    def step():
        H.check(H.lib().ihip_enqueue_paged_slots(
            ctx.h, bufs["past"].ptr, 0, n, bufs["table"].ptr, width, 4, bufs["ring"].ptr, len(ring),
            bufs["ends"].ptr, bufs["ends"].ptr, o.ptr, bufs["past"].ptr, q.ptr, s.ptr, n, f.ptr))

    H.check(H.lib().ihip_capture_begin(ctx.h))
    step()
    H.check(H.lib().ihip_capture_end(ctx.h, 9))
    for _ in range(12):
        want = R.slots(past, None, table, 4, ring, ends, n)
        H.check(H.lib().ihip_graph_launch(ctx.h, 9))
        for k, b, dt in (("table", bufs["table"], np.int32), ("ring", bufs["ring"], np.int32),
                         ("ends", bufs["ends"], np.int64), ("lengths", bufs["past"], np.int32),
                         ("slots", s, np.int32), ("positions", q, np.int32),
                         ("offsets", o, np.int32)):
            assert np.array_equal(b.download(dt, want[k].size), want[k].ravel()), k
        past, table, ring, ends = (want[k] for k in ("lengths", "table", "ring", "ends"))


# -------------------------------------------------------------------- qkrope
def pool_of(rng, shape, dtype):
    return R.pack(rng.standard_normal(shape), dtype)


def strides_of(layout, page_size, kvh, hd):
    """(page, slot, head) strides and the numpy axes of [pages, page_size, kv_heads, hd]."""
    if layout == "heads":
        return (page_size * kvh * hd, hd, page_size * hd), (0, 2, 1, 3)
    return (0, 0, 0), (0, 1, 2, 3)


def pages_struct(dk, dv, pages, page_size, kvh, hd, dtype, layout="tokens"):
    st, _ = strides_of(layout, page_size, kvh, hd)
    return H.Pages(k=dk, v=dv, pages=pages, page_stride=st[0], slot_stride=st[1], head_stride=st[2],
                   page_size=page_size, kv_heads=kvh, head_dim=hd, dtype=CODE[dtype])


@pytest.mark.parametrize("hd,heads,kvh,dims,inter,norm,dtype,layout,pad,most", [
    (128, 32, 4, 0, 0, True, "f16", "tokens", 0, 5000), (128, 16, 8, 128, 1, False, "bf16", "tokens", 0, 131072),
    (64, 64, 8, 64, 0, False, "f16", "heads", 0, 40000), (256, 8, 2, 64, 0, True, "f32", "tokens", 8, 3000),
    (256, 8, 2, 64, 1, True, "bf16", "heads", 4, 3000), (512, 16, 2, 128, 0, True, "f16", "tokens", 0, 9000),
    (80, 4, 4, 20, 0, False, "f32", "tokens", 0, 2 ** 31 - 1), (80, 4, 2, 10, 1, True, "f16", "tokens", 0, 100),
    (96, 12, 12, 96, 0, True, "bf16", "tokens", 3, 800), (8, 2, 1, 2, 0, True, "f32", "tokens", 1, 60),
    (8, 1, 1, 8, 1, False, "f16", "heads", 0, 60), (72, 3, 1, 6, 0, False, "f16", "tokens", 0, 70),
    (128, 32, 4, -1, 0, True, "f16", "tokens", 0, 500)])
@pytest.mark.parametrize("rows", [1, 5, 67])
def test_qkrope(ctx, dev, hd, heads, kvh, dims, inter, norm, dtype, layout, pad, most, rows):
    rng = np.random.default_rng(hd * heads + rows + inter)
    ps = int(rng.choice([1, 7, 16]))
    pages = rows // ps + 3
    width = (heads + 2 * kvh) * hd + pad
    x = rng.standard_normal((rows, width)).astype(np.float32) * 3
    qn, kn = (rng.standard_normal(hd).astype(np.float32) + 1 for _ in range(2))
    positions = rng.integers(0, most, rows).astype(np.int32)
    slots = rng.permutation(pages * ps)[:rows].astype(np.int32)
    if rows > 4:
        positions[1], slots[2], slots[3] = -1, -1, pages * ps
    st, axes = strides_of(layout, ps, kvh, hd)
    k0, v0 = (pool_of(rng, (pages, ps, kvh, hd), dtype) for _ in range(2))
    lay = [np.ascontiguousarray(a.transpose(axes)) for a in (k0, v0)]
    dk, dv = (dev.out(a.nbytes) for a in lay)
    dk.upload(lay[0]), dv.upload(lay[1])
    rope, freq, scale, d = None, None, 1.0, dims if dims > 0 else hd
    if dims >= 0:
        scale = 1.25 if inter else 0.0
        freq = (1.0 / 10000.0 ** (np.arange(0, d, 2) / d)).astype(np.float32)
        rope = H.Rope(freq=dev(freq), dims=dims, interleaved=inter, scale=scale)
    dx, dy = dev.out(x.nbytes), dev.out(rows * heads * hd * 4)
    dx.upload(x)
    pool = pages_struct(dk.ptr, dv.ptr, pages, ps, kvh, hd, dtype, layout)

    dqn, dkn = (dev(qn), dev(kn)) if norm else (0, 0)
    dpos, dslots = dev(positions), dev(slots)

    def call(out):
        q = dx.ptr
        return H.lib().ihip_enqueue_paged_qkrope(
            ctx.h, q, width, q + 4 * heads * hd, width, q + 4 * (heads + kvh) * hd, width, rows, heads,
            dqn, dkn, 1e-6, C.byref(rope) if rope is not None else None,
            dpos, dslots, C.byref(pool), out)

    H.check(call(dy.ptr), "qkrope")
    q, k, v = np.split(x[:, :width - pad].reshape(rows, -1, hd), (heads, heads + kvh), 1)
    live = positions >= 0
    want_q = R.rope(q, qn if norm else None, 1e-6, freq, d, inter, scale or 1.0, positions)
    want_k = R.rope(k, kn if norm else None, 1e-6, freq, d, inter, scale or 1.0, positions)
    got = dy.download(np.float32, want_q.size).reshape(want_q.shape)

    def close(g, w, x, step):
        # one rounding of a double result; the double sums stay below 1e-13 of a pair's values
        size = np.abs(w).max(-1, keepdims=True) + np.abs(x).max(-1, keepdims=True)
        assert np.all(np.abs(g - w) <= step * np.abs(w) * (1 + 2.0 ** -10) + 1e-12 * size + 2.0 ** -25 * (step > U)), \
            np.abs(g - w).max()

    close(got[live], want_q[live], q[live], U)
    assert (got[~live].view(np.uint8) == 0x5A).all()
    for raw, old, want, src in ((dk, k0, want_k, k), (dv, v0, v.astype(np.float64), v)):
        new = raw.download(old.dtype, old.size).reshape(lay[0].shape).transpose(axes)
        flat, was = new.reshape(pages * ps, kvh, hd), old.reshape(pages * ps, kvh, hd)
        stored = live & (slots >= 0) & (slots < pages * ps)
        close(R.unpack(flat[slots[stored]], dtype), want[stored], src[stored], R.HALF_STEP[dtype])
        rest = np.ones(pages * ps, bool)
        rest[slots[stored]] = False
        assert np.array_equal(flat[rest], was[rest])
    # k and v of the rows are left, q too unless it is the output
    assert np.array_equal(dx.download(np.float32, x.size).reshape(x.shape), x)
    H.check(call(0), "in place")
    after = dx.download(np.float32, x.size).reshape(x.shape)
    assert np.array_equal(after[:, heads * hd:], x[:, heads * hd:])
    assert np.array_equal(after[live][:, :heads * hd].reshape(-1), got[live].reshape(-1))
    assert np.array_equal(after[~live], x[~live])


# ----------------------------------------------------------------- attention
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, -1, 127, 128, 129, 257, 1000]


def attention_case(ctx, dev, rng, dtype, hd, heads, kvh, ps, lengths, window=0, sinks=False, scale=0.0,
                   layout="tokens", pad=0, change=None, width=None):
    lengths = np.array(lengths, np.int32)
    have = -(-np.maximum(lengths, 0) // ps)
    n, pages = len(lengths), int(have.sum()) + 3
    width = width or max(1, int(have.max()) + 1)
    order = rng.permutation(pages)
    table = rng.integers(-2 ** 31, 2 ** 31, (n, width)).astype(np.int32)  # nobody's pages
    at = 0
    for s in range(n):
        table[s, :have[s]] = order[at:at + have[s]]
        at += have[s]
    k, v = (rng.standard_normal((pages, ps, kvh, hd)) for _ in range(2))
    q = rng.standard_normal((n, heads * hd + pad)).astype(np.float32)
    sk = (rng.standard_normal(heads) * 2).astype(np.float32) if sinks else None
    # what no sequence holds: NaN and infinities
    held = np.zeros((pages, ps), bool)
    for s in range(n):
        for p, t in R.keys_of(table[s], lengths[s], 0, ps, pages):
            held[p, t] = True
    k[~held], v[~held] = np.nan, np.inf
    if change:
        change(q, k, v, table, lengths)
    kr, vr = R.pack(k, dtype), R.pack(v, dtype)
    _, axes = strides_of(layout, ps, kvh, hd)
    dk, dv = (dev(np.ascontiguousarray(a.transpose(axes))) for a in (kr, vr))
    pool = pages_struct(dk, dv, pages, ps, kvh, hd, dtype, layout)
    y = dev.out(n * heads * hd * 4)
    H.check(H.lib().ihip_enqueue_paged_attention(
        ctx.h, dev(q), heads * hd + pad if pad else 0, C.byref(pool), dev(table), width, dev(lengths),
        y.ptr, n, heads, window, dev(sk) if sinks else 0, scale), "attention")
    got = y.download(np.float32, n * heads * hd).reshape(n, heads, hd)
    q64 = q[:, :heads * hd].reshape(n, heads, hd).astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol = R.attention(q64, R.unpack(kr, dtype), R.unpack(vr, dtype), table, lengths, ps, window,
                                sk, scale)
    assert (got[lengths < 0].view(np.uint8) == 0x5A).all()
    return got[lengths >= 0], want[lengths >= 0], tol[lengths >= 0], lengths[lengths >= 0]


def assert_close(got, want, tol, lengths=None):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), np.abs(got - want)[bad][:5], tol[bad][:5])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd,heads,kvh,ps", [(128, 32, 4, 16), (64, 64, 8, 32), (256, 8, 2, 64), (512, 16, 2, 16),
                                             (96, 12, 12, 7), (80, 32, 2, 1), (8, 3, 1, 24), (128, 48, 2, 256),
                                             (136, 17, 1, 100), (512, 2, 2, 1)])
def test_attention(ctx, dev, dtype, hd, heads, kvh, ps):
    rng = np.random.default_rng(hd + heads + ps)
    assert_close(*attention_case(ctx, dev, rng, dtype, hd, heads, kvh, ps, LENGTHS))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("window,sinks,scale,layout,pad", [
    (1, False, 0.0, "tokens", 0), (16, True, 0.0, "heads", 8), (33, False, 0.3, "tokens", 3),
    (128, True, 0.0, "tokens", 0), (10 ** 6, True, 0.05, "heads", 0), (0, True, 2.0, "heads", 64)])
def test_attention_windows_sinks_strides(ctx, dev, dtype, window, sinks, scale, layout, pad):
    rng = np.random.default_rng(window + pad)
    assert_close(*attention_case(ctx, dev, rng, dtype, 64, 8, 2, 16, LENGTHS + [300, 700], window, sinks, scale,
                                 layout, pad))


@pytest.mark.parametrize("dtype,hd,heads,kvh,ps,lengths", [
    ("f16", 128, 8, 1, 16, [20000]), ("bf16", 64, 4, 2, 100, [9000, 1, 3]), ("f32", 256, 2, 1, 33, [5000]),
    ("f16", 512, 4, 1, 64, [4000, 2]), ("f16", 128, 32, 4, 16, [1152]), ("f16", 64, 40, 1, 8, [1, 6000, 0, 77] * 3),
    ("bf16", 128, 16, 8, 16, list(range(1, 200, 3)))])
def test_attention_split_over_the_length(ctx, dev, dtype, hd, heads, kvh, ps, lengths):
    """Long sequences beside short ones: the blocks' parts of a sequence joined."""
    rng = np.random.default_rng(len(lengths) + hd)
    assert_close(*attention_case(ctx, dev, rng, dtype, hd, heads, kvh, ps, lengths))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_with_long_streams(ctx, dev, dtype):
    """Tiles enough for one block a CU, a block's pieces of several heads and sequences."""
    rng = np.random.default_rng(17)
    assert_close(*attention_case(ctx, dev, rng, dtype, 8, 64, 64, 64, [8300, 8192, 0, 8400, 8250, 30]))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_large_scores_and_queries(ctx, dev, dtype):
    """Scores far apart, a query of tiny and one of huge values, equal keys."""
    def change(q, k, v, table, lengths):
        q[1] *= 300
        q[2] *= 1e-30
        q[3] *= 1e4
        q[4] = 0
        q[5, :64] *= 1e-6  # a head whose first values are tiny
        for j in range(40):
            k[table[0][j // 16], j % 16] = k[table[0][0], 0]
        k[table[3][0], :] *= 100
        v[table[2][0], 3] *= 6e4 / 4

    rng = np.random.default_rng(77)
    assert_close(*attention_case(ctx, dev, rng, dtype, 128, 8, 2, 16, [40, 130, 65, 70, 90, 33], change=change))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_pages_that_are_not_there(ctx, dev, dtype):
    """Table entries outside the pool hide their keys, all of a sequence's among them; a length
    beyond the table is cut to it."""
    def change(q, k, v, table, lengths):
        table[0, 1], table[0, 3] = -1, 2 ** 31 - 1
        table[1, :] = -5
        table[2, 0] = len(k)
        lengths[3] = 2 ** 31 - 1
        table[3, 2:] = -1

    rng = np.random.default_rng(5)
    got, want, tol, _ = attention_case(ctx, dev, rng, dtype, 128, 8, 2, 16, [100, 60, 30, 33], sinks=True,
                                       change=change, width=9)
    # (the last page of sequence 3 holds one key of its own and NaN behind it, now seen)
    assert_close(got[:3], want[:3], tol[:3])
    assert np.isnan(got[3]).all() or np.isfinite(want[3]).all()
    assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_infinities_and_nan(ctx, dev, dtype):
    """A NaN or an infinity reaches the rows, heads and dimensions that see it, and no others."""
    def change(q, k, v, table, lengths):
        v[table[1][0], 3, 1, 5] = np.inf
        v[table[2][1], 0, 0, 7] = np.nan
        k[table[3][0], 2, 0, 4] = np.nan
        k[table[4][2], 9, 1, 0] = np.inf
        q[4, :] = np.abs(q[4, :])
        q[5, 3 * 128 + 1] = np.inf
        k[table[6][0], 1, 0, 3] = -np.inf
        q[6, :] = np.abs(q[6, :])

    rng = np.random.default_rng(6)
    got, want, tol, _ = attention_case(ctx, dev, rng, dtype, 128, 8, 2, 16, [50, 50, 200, 40, 90, 64, 48],
                                       change=change)
    assert_close(got[0], want[0], tol[0])
    inf = np.zeros((8, 128), bool)
    inf[4:, 5] = True
    assert (got[1][inf] == np.inf).all()
    assert_close(got[1][~inf], want[1][~inf], tol[1][~inf])
    nan = np.zeros((8, 128), bool)
    nan[:4, 7] = True
    assert np.isnan(got[2][nan]).all()
    assert_close(got[2][~nan], want[2][~nan], tol[2][~nan])
    assert np.isnan(got[3][:4]).all()  # (its KV head's group)
    assert_close(got[3][4:], want[3][4:], tol[3][4:])
    assert np.isnan(got[4][4:]).all()  # a score of infinity
    assert_close(got[4][:4], want[4][:4], tol[4][:4])
    assert np.isnan(got[5][3]).all()
    others = np.arange(8) != 3
    assert_close(got[5][others], want[5][others], tol[5][others])
    # a score of -infinity is a key of weight 0
    assert np.isfinite(got[6]).all()


def test_attention_beyond_32_bits(ctx, dev):
    """Pages whose values lie past 2^32 bytes and past 2^31 values of the pool."""
    hd, kvh, ps, pages = 128, 2, 16, 3
    stride = (1 << 30) + 64
    rng = np.random.default_rng(8)
    big = ctx.alloc((2 * stride + ps * kvh * hd * 4) * 4)
    try:
        k, v = (np.ascontiguousarray(a) for a in rng.standard_normal((2, pages, ps, kvh, hd)).astype(np.float32))
        half = ps * kvh * hd  # the values behind the keys of the same page
        for p in range(pages):
            H.check(H.lib().ihip_upload(ctx.h, big.ptr + 4 * p * stride, k.ctypes.data + p * k[p].nbytes, k[p].nbytes))
            H.check(H.lib().ihip_upload(ctx.h, big.ptr + 4 * (p * stride + half), v.ctypes.data + p * v[p].nbytes, v[p].nbytes))
        pool = H.Pages(k=big.ptr, v=big.ptr + 4 * half, pages=pages, page_stride=stride, page_size=ps, kv_heads=kvh,
                       head_dim=hd, dtype=H.F32)
        q = rng.standard_normal((2, 4, hd)).astype(np.float32)
        table, lengths = np.array([[2, 0, 1], [1, 2, 0]], np.int32), np.array([41, 20], np.int32)
        y = dev.out(q.nbytes)
        H.check(H.lib().ihip_enqueue_paged_attention(ctx.h, dev(q), 0, C.byref(pool), dev(table), 3, dev(lengths),
                                                     y.ptr, 2, 4, 0, 0, 0.0), "attention")
        got = y.download(np.float32, q.size).reshape(q.shape)
        want, tol = R.attention(q.astype(np.float64), k.astype(np.float64), v.astype(np.float64), table, lengths, ps)
        assert_close(got, want, tol)
        # and stored there
        x = rng.standard_normal((2, 8, hd)).astype(np.float32)
        slots = np.array([2 * ps + 15, ps + 3], np.int32)
        dx = dev(x)
        H.check(H.lib().ihip_enqueue_paged_qkrope(
            ctx.h, dx, 8 * hd, dx + 4 * 4 * hd, 8 * hd, dx + 4 * 6 * hd, 8 * hd, 2, 4, 0, 0, 0.0, None,
            dev(np.array([1, 2], np.int32)), dev(slots), C.byref(pool), 0), "store")
        for r, s in enumerate(slots.tolist()):
            for off, part in ((0, x[r, 4:6]), (half, x[r, 6:8])):
                back = np.empty((kvh, hd), np.float32)
                H.check(H.lib().ihip_download(ctx.h, H._p(back), big.ptr + 4 * (s // ps * stride + off +
                                                                              s % ps * kvh * hd), back.nbytes))
                assert np.array_equal(back, part)
    finally:
        ctx.sync()
        big.free()


def test_attention_repeats_bit_for_bit(ctx, dev):
    rng = np.random.default_rng(12)
    runs = []
    for _ in range(3):
        rng = np.random.default_rng(12)
        runs.append(attention_case(ctx, dev, rng, "f16", 128, 16, 2, 16, [3000, 5, 900, 64, 2000])[0])
    assert all(np.array_equal(runs[0].view(np.uint32), r.view(np.uint32)) for r in runs[1:])


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype,graph", [("f16", False), ("f16", True), ("bf16", True), ("f32", True)])
def test_decode_steps_together(ctx, dev, dtype, graph):
    """Sequences of a batch over several steps: prompts of unlike lengths stored, then single
    tokens, one sequence ending and an empty place, each step planned, stored and attended on the
    device alone; the attention against the cache's own values in 64 bits."""
    hd, heads, kvh, ps, width, n, pages = 64, 8, 2, 4, 16, 5, 48
    rng = np.random.default_rng(21)
    past = np.array([0, 0, 0, -1, 0], np.int32)
    prompt = np.array([9, 1, 30, 0, 17], np.int32)
    table = np.full((n, width), -1, np.int32)
    ring, ends = rng.permutation(pages).astype(np.int32), np.array([0, pages], np.int64)
    freq = (1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd)).astype(np.float32)
    rope = H.Rope(freq=dev(freq))
    cap = 64
    es = 4 if dtype == "f32" else 2
    pool_bytes = pages * ps * kvh * hd * es
    dk, dv = dev.out(pool_bytes, 0xFF), dev.out(pool_bytes, 0xFF)  # NaN everywhere
    pool = pages_struct(dk.ptr, dv.ptr, pages, ps, kvh, hd, dtype)
    b = {}
    for name, a in dict(past=past, table=table, ring=ring, ends=ends).items():
        b[name] = dev.out(a.nbytes)
        b[name].upload(a)
    dcount, dx = dev.out(4 * n), dev.out(cap * (heads + 2 * kvh) * hd * 4)
    offs, pos, slots, failed = dev.out(4 * n + 4), dev.out(4 * cap), dev.out(4 * cap), dev.out(4)
    y = dev.out(n * heads * hd * 4)
    row = (heads + 2 * kvh) * hd

    def plan(rows):
        H.check(H.lib().ihip_enqueue_paged_slots(
            ctx.h, b["past"].ptr, dcount.ptr, n, b["table"].ptr, width, ps, b["ring"].ptr, pages,
            b["ends"].ptr, b["ends"].ptr, offs.ptr, b["past"].ptr, pos.ptr, slots.ptr, rows, failed.ptr))

    def store(rows):
        q = dx.ptr
        H.check(H.lib().ihip_enqueue_paged_qkrope(
            ctx.h, q, row, q + 4 * heads * hd, row, q + 4 * (heads + kvh) * hd, row, rows, heads, 0, 0, 0.0,
            C.byref(rope), pos.ptr, slots.ptr, C.byref(pool), 0))

    def attend():
        H.check(H.lib().ihip_enqueue_paged_attention(
            ctx.h, dx.ptr, row, C.byref(pool), b["table"].ptr, width, b["past"].ptr, y.ptr, n, heads, 0, 0, 0.0))

    dcount.upload(prompt)
    dx.upload(rng.standard_normal((cap, row)).astype(np.float32))
    plan(cap), store(cap)
    lengths = np.where(past < 0, -1, prompt)
    if graph:
        H.check(H.lib().ihip_capture_begin(ctx.h))
        plan(n), store(n), attend()
        H.check(H.lib().ihip_capture_end(ctx.h, 10))
    for step in range(6):
        # every place of the batch brings its row; sequence 2 ends at step 3
        count = np.array([1, 1, -1 if step == 3 else 1, 1, 1], np.int32)
        dcount.upload(count)
        # rows in the batch's order: live sequences' rows come first to last
        x = rng.standard_normal((n, row)).astype(np.float32)
        dx.upload(x)
        y.upload(np.full(n * heads * hd * 4, 0x5A, np.uint8))
        if graph:
            H.check(H.lib().ihip_graph_launch(ctx.h, 10))
        else:
            plan(n), store(n), attend()
        lengths = np.where((lengths < 0) | (count < 0), -1, lengths + 1)
        assert np.array_equal(b["past"].download(np.int32, n), lengths), step
        assert failed.download(np.int32, 1)[0] == 0
        t = b["table"].download(np.int32, n * width).reshape(n, width)
        live = lengths >= 0
        assert len(set(t[live][t[live] >= 0].tolist())) == sum(-(-l // ps) for l in lengths[live])
        raw = [d.download(np.uint8, pool_bytes).view({"f32": np.float32, "f16": np.float16,
                                                     "bf16": np.uint16}[dtype]).reshape(pages, ps, kvh, hd)
               for d in (dk, dv)]
        q = dx.download(np.float32, n * row).reshape(n, row)
        # (the attention reads row s of sequence s)
        with np.errstate(invalid="ignore"):
            want, tol = R.attention(q[:, :heads * hd].reshape(n, heads, hd).astype(np.float64),
                                    R.unpack(raw[0], dtype), R.unpack(raw[1], dtype), t, lengths, ps)
        got = y.download(np.float32, n * heads * hd).reshape(n, heads, hd)
        assert_close(got[live], want[live], tol[live])
        assert (got[~live].view(np.uint8) == 0x5A).all()
        # the step's keys are the rows': rotated at their positions, in their slots
        p, s = pos.download(np.int32, n), slots.download(np.int32, n)
        m = int(live.sum())
        assert (p[m:] == -1).all() and np.array_equal(p[:m], lengths[live] - 1)
        kk = R.rope(x[:m, heads * hd:(heads + kvh) * hd].reshape(m, kvh, hd), None, 0, freq, hd, 0, 1.0, p[:m])
        have = R.unpack(raw[0].reshape(-1, kvh, hd)[s[:m]], dtype)
        assert np.all(np.abs(have - kk) <= R.HALF_STEP[dtype] * np.abs(kk) * 1.01 + 1e-6)


def test_two_contexts(dev, ctx):
    """A second context's calls between the first's, on their own streams."""
    rng = np.random.default_rng(31)
    with H.Context(0) as other:
        def dev2(a):
            return other.array(a).ptr

        dev2.out = lambda n, fill=0x5A: other.array(np.full(n, fill, np.uint8))
        for i in range(3):
            assert_close(*attention_case(ctx, dev, rng, "f16", 128, 16, 2, 16, [1500, 3, 700])[:3])
            assert_close(*attention_case(other, dev2, rng, "f16", 128, 16, 2, 16, [900, 2500])[:3])


def test_first_calls_captured():
    """The first calls of a context, captured before any kernel of theirs has run; two graphs of
    one context share its workspaces, replayed in turn over other lengths."""
    rng = np.random.default_rng(51)
    n, heads, kvh, hd, ps, pages = 6, 16, 2, 128, 16, 400
    with H.Context(0) as c:
        k, v = (R.pack(rng.standard_normal((pages, ps, kvh, hd)), "f16") for _ in range(2))
        dk, dv = c.array(k), c.array(v)
        pool = pages_struct(dk.ptr, dv.ptr, pages, ps, kvh, hd, "f16")
        table = rng.permutation(pages)[:n * 60].reshape(n, 60).astype(np.int32)
        q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        x = rng.standard_normal((3, 40000)).astype(np.float32)
        dt, dq, dx = c.array(table), c.array(q), c.array(x)
        lens = [c.array(np.zeros(n, np.int32)) for _ in range(2)]
        ys = [c.alloc(q.nbytes) for _ in range(2)]
        top = [[c.alloc(4 * 3 * 8) for _ in range(2)] for _ in range(2)]
        for g in range(2):
            H.check(H.lib().ihip_capture_begin(c.h))
            H.check(H.lib().ihip_enqueue_paged_attention(
                c.h, dq.ptr, 0, C.byref(pool), dt.ptr, 60, lens[g].ptr, ys[g].ptr, n, heads, 0, 0, 0.0))
            H.check(H.lib().ihip_enqueue_logprobs(c.h, dx.ptr, 3, 40000, 0, 0, 0, 0, 8, top[g][0].ptr, top[g][1].ptr))
            H.check(H.lib().ihip_capture_end(c.h, g))
        for i in range(5):
            ln = [rng.integers(0, 960, n).astype(np.int32) for _ in range(2)]
            for g in range(2):
                lens[g].upload(ln[g])
            for g in range(2):
                H.check(H.lib().ihip_graph_launch(c.h, g))
            for g in range(2):
                got = ys[g].download(np.float32, q.size).reshape(q.shape)
                want, tol = R.attention(q.astype(np.float64), R.unpack(k, "f16"), R.unpack(v, "f16"), table, ln[g], ps)
                assert_close(got, want, tol)
                ids = top[g][0].download(np.int32, 24).reshape(3, 8)
                assert np.array_equal(ids, np.stack([R.order(r)[:8] for r in x]))
            # an eager call between the replays
            H.check(H.lib().ihip_enqueue_paged_attention(
                c.h, dq.ptr, 0, C.byref(pool), dt.ptr, 60, lens[0].ptr, ys[1].ptr, n, heads, 0, 0, 0.0))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_many_short_sequences(ctx, dev, dtype):
    """More sequences than a wave scans at once, empty places and empty rows among them."""
    rng = np.random.default_rng(61)
    lengths = rng.integers(-1, 40, 700)
    lengths[rng.random(700) < 0.3] = 0
    assert_close(*attention_case(ctx, dev, rng, dtype, 64, 2, 1, 8, lengths.tolist()))


def test_attention_of_nobody(ctx, dev):
    """No sequence has a key: zeros and rows left alone, nothing else."""
    rng = np.random.default_rng(62)
    got, want, tol, lengths = attention_case(ctx, dev, rng, "bf16", 128, 8, 2, 16, [0, -1, 0, -5, 0])
    assert (got == 0).all() and len(got) == 3


def test_attention_shares_pages(ctx, dev):
    """Two sequences over the same pages (a common prompt), unlike lengths."""
    def change(q, k, v, table, lengths):
        table[1, :4] = table[0, :4]

    rng = np.random.default_rng(63)
    assert_close(*attention_case(ctx, dev, rng, "f16", 128, 8, 2, 16, [90, 60], change=change))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_by_rows(ctx, dev, dtype):
    """Sequences whose rows are a step's: the last row of each, none of an empty or ended place,
    none beyond the rows there are."""
    rng = np.random.default_rng(71)
    n, heads, kvh, hd, ps, width, rows = 9, 8, 2, 128, 16, 12, 14
    counts = np.array([1, 0, 3, 1, 0, 5, 2, 1, 4])  # the last ends beyond the rows
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    lengths = np.array([40, 33, 0, 150, -1, 90, -1, 77, 60], np.int32)
    pages = n * width
    k, v = (R.pack(rng.standard_normal((pages, ps, kvh, hd)), dtype) for _ in range(2))
    table = rng.permutation(pages).reshape(n, width).astype(np.int32)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    pool = pages_struct(dev(k), dev(v), pages, ps, kvh, hd, dtype)
    y = dev.out(q.nbytes)
    H.check(H.lib().ihip_enqueue_paged_attention_at(
        ctx.h, dev(q), 0, C.byref(pool), dev(table), width, dev(lengths), dev(offsets), rows, y.ptr, n, heads, 0, 0,
        0.0))
    got = y.download(np.float32, q.size).reshape(q.shape)
    written = np.zeros(rows, bool)
    for s in range(n):
        r = offsets[s + 1] - 1
        if counts[s] == 0 or r >= rows or lengths[s] < 0:
            continue
        written[r] = True
        want, tol = R.attention(q[r:r + 1].astype(np.float64), R.unpack(k, dtype), R.unpack(v, dtype), table[s:s + 1],
                                lengths[s:s + 1], ps)
        assert_close(got[r], want[0], tol[0])
    assert written.tolist() == [i in (0, 3, 4, 9, 12) for i in range(rows)]
    assert (got[~written].view(np.uint8) == 0x5A).all()


def test_decode_steps_by_rows(ctx, dev):
    """Replayed steps of a batch with empty places: each sequence's query is its own row of the
    step, its output there too, against a host model that keeps every sequence's keys apart."""
    hd, heads, kvh, ps, width, n, pages = 64, 4, 2, 4, 12, 6, 60
    rng = np.random.default_rng(81)
    past = np.array([0, -1, 0, 0, -1, 0], np.int32)
    row = (heads + 2 * kvh) * hd
    b = {}
    for name, a in dict(past=past, count=np.zeros(n, np.int32), table=np.full((n, width), -1, np.int32),
                        ring=rng.permutation(pages).astype(np.int32), ends=np.array([0, pages], np.int64)).items():
        b[name] = dev.out(a.nbytes)
        b[name].upload(a)
    kc, vc = dev.out(pages * ps * kvh * hd * 4, 0xFF), dev.out(pages * ps * kvh * hd * 4, 0xFF)
    pool = pages_struct(kc.ptr, vc.ptr, pages, ps, kvh, hd, "f32")
    x, y = dev.out(n * row * 4), dev.out(n * heads * hd * 4)
    offs, pos, slots, failed = (dev.out(4 * m) for m in (n + 1, n, n, 1))
    H.check(H.lib().ihip_capture_begin(ctx.h))
    H.check(H.lib().ihip_enqueue_paged_slots(
        ctx.h, b["past"].ptr, b["count"].ptr, n, b["table"].ptr, width, ps, b["ring"].ptr, pages, b["ends"].ptr,
        b["ends"].ptr, offs.ptr, b["past"].ptr, pos.ptr, slots.ptr, n, failed.ptr))
    H.check(H.lib().ihip_enqueue_paged_qkrope(
        ctx.h, x.ptr, row, x.ptr + 4 * heads * hd, row, x.ptr + 4 * (heads + kvh) * hd, row, n, heads, 0, 0, 0.0, None,
        pos.ptr, slots.ptr, C.byref(pool), 0))
    H.check(H.lib().ihip_enqueue_paged_attention_at(
        ctx.h, x.ptr, row, C.byref(pool), b["table"].ptr, width, b["past"].ptr, offs.ptr, n, y.ptr, n, heads, 0, 0, 0.0))
    H.check(H.lib().ihip_capture_end(ctx.h, 12))
    keys = {s: ([], []) for s in range(n) if past[s] >= 0}
    for step in range(20):
        count = np.array([1, 1, step % 2, 1, 1, -1 if step == 11 else 1], np.int32)
        data = rng.standard_normal((n, row)).astype(np.float32)
        b["count"].upload(count), x.upload(data)
        H.check(H.lib().ihip_graph_launch(ctx.h, 12))
        if step == 11:
            del keys[5]
        got = y.download(np.float32, n * heads * hd).reshape(n, heads, hd)
        assert failed.download(np.int32, 1)[0] == 0
        r = 0
        for s in sorted(keys):
            if not count[s]:
                continue
            q, kk, vv = np.split(data[r].reshape(-1, hd), (heads, heads + kvh))
            keys[s][0].append(kk), keys[s][1].append(vv)
            k64, v64 = (np.array(a).astype(np.float64)[None] for a in keys[s])
            want, tol = R.attention(q[None].astype(np.float64), k64, v64, np.array([[0]]), [k64.shape[1]], k64.shape[1])
            assert_close(got[r], want[0], tol[0])
            r += 1

"""8-bit pages on the device against their definition in 64 bits: rows quantized as they
are stored, read back, and attended (paged_ref.py's attention of codes times scales)."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_ref as R
from test_gpu_paged import LENGTHS, assert_close, ctx, dev, strides_of  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
U = R.U


def q8_pool(ptrs, pages, ps, kvh, hd, layout="tokens"):
    st, _ = strides_of(layout, ps, kvh, hd)
    k, v, ks, vs = ptrs
    return H.Pages(k=k, v=v, pages=pages, page_stride=st[0], slot_stride=st[1], head_stride=st[2], page_size=ps,
                   kv_heads=kvh, head_dim=hd, dtype=H.Q8_HEAD, k_scale=ks, v_scale=vs)


def order(layout):
    return (0, 2, 1, 3) if layout == "heads" else (0, 1, 2, 3)


# --------------------------------------------------------------------- store
@pytest.mark.parametrize("hd,heads,kvh,dims,inter,norm,layout,pad,most", [
    (128, 32, 4, 0, 0, True, "tokens", 0, 5000), (128, 16, 8, 128, 1, False, "heads", 0, 131072),
    (64, 64, 8, 64, 0, False, "heads", 0, 40000), (256, 8, 2, 64, 0, True, "tokens", 8, 3000),
    (512, 16, 2, 128, 0, True, "tokens", 0, 9000), (80, 4, 4, 20, 0, False, "tokens", 0, 2 ** 31 - 1),
    (80, 4, 2, 10, 1, True, "heads", 0, 100), (96, 12, 12, 96, 0, True, "tokens", 3, 800),
    (16, 3, 1, 6, 0, False, "tokens", 1, 70), (16, 1, 1, 16, 1, True, "heads", 0, 60),
    (128, 32, 4, -1, 0, True, "tokens", 0, 500)])
@pytest.mark.parametrize("rows", [1, 5, 67])
def test_store(ctx, dev, hd, heads, kvh, dims, inter, norm, layout, pad, most, rows):
    rng = np.random.default_rng(hd * heads + rows + inter)
    ps = int(rng.choice([1, 7, 16]))
    pages, width = rows // ps + 3, (heads + 2 * kvh) * hd + pad
    x = rng.standard_normal((rows, width)).astype(np.float32) * 3
    x[0, heads * hd:(heads + 1) * hd] = 0  # a head of zeros
    qn, kn = (rng.standard_normal(hd).astype(np.float32) + 1 for _ in range(2))
    positions = rng.integers(0, most, rows).astype(np.int32)
    slots = rng.permutation(pages * ps)[:rows].astype(np.int32)
    if rows > 4:
        positions[1], slots[2], slots[3] = -1, -1, pages * ps
    shape = [(pages, ps, kvh, hd)[i] for i in order(layout)]
    old = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
    old += [rng.random(shape[:3]).astype(np.float32) for _ in range(2)]
    bufs = [dev.out(a.nbytes) for a in old]
    for b, a in zip(bufs, old):
        b.upload(a)
    rope, freq, scale, d = None, None, 1.0, dims if dims > 0 else hd
    if dims >= 0:
        scale = 1.25 if inter else 0.0
        freq = (1.0 / 10000.0 ** (np.arange(0, d, 2) / d)).astype(np.float32)
        rope = H.Rope(freq=dev(freq), dims=dims, interleaved=inter, scale=scale)
    pool = q8_pool([b.ptr for b in bufs], pages, ps, kvh, hd, layout)
    q, y = dev(x), dev.out(rows * heads * hd * 4)
    H.check(H.lib().ihip_enqueue_paged_qkrope(
        ctx.h, q, width, q + 4 * heads * hd, width, q + 4 * (heads + kvh) * hd, width, rows, heads,
        dev(qn) if norm else 0, dev(kn) if norm else 0, 1e-6, C.byref(rope) if rope is not None else None,
        dev(positions), dev(slots), C.byref(pool), y.ptr), "store")
    qq, k, v = np.split(x[:, :width - pad].reshape(rows, -1, hd), (heads, heads + kvh), 1)
    args = (1e-6, freq, d, inter, scale or 1.0, positions)
    live = positions >= 0
    got_q, want_q = y.download(np.float32, qq.size).reshape(qq.shape), R.rope(qq, qn if norm else None, *args)
    size = np.abs(want_q).max(-1, keepdims=True) + np.abs(qq).max(-1, keepdims=True)
    assert np.all(np.abs(got_q - want_q)[live] <= (U * np.abs(want_q) * 1.001 + 1e-12 * size)[live])
    stored = live & (slots >= 0) & (slots < pages * ps)
    rest = np.ones(pages * ps, bool)
    rest[slots[stored]] = False
    for i, want in ((0, R.rope(k, kn if norm else None, *args)), (1, v.astype(np.float64))):
        back = np.argsort(order(layout))
        codes = bufs[i].download(np.int8, old[i].size).reshape(shape).transpose(back).reshape(-1, kvh, hd)
        sc = bufs[i + 2].download(np.float32, old[i + 2].size).reshape(shape[:3]).transpose(back[:3]).reshape(-1, kvh)
        was = old[i].transpose(back).reshape(-1, kvh, hd), old[i + 2].transpose(back[:3]).reshape(-1, kvh)
        assert np.array_equal(codes[rest], was[0][rest]) and np.array_equal(sc[rest], was[1][rest])
        c, s, w = codes[slots[stored]].astype(np.float64), sc[slots[stored]].astype(np.float64), want[stored]
        # the scale is one rounding of a quotient of doubles, a value half a step off (the
        # doubles' own error, 1e-12 of the head, moves the border)
        top = np.abs(w).max(-1)
        assert np.all(np.abs(s - top / 127) <= top / 127 * (U * 1.001 + 1e-12))
        assert np.all(np.abs(c * s[..., None] - w) <= s[..., None] * (0.5 + 1e-9) + 1e-12 * top[..., None])


def test_store_borders(ctx, dev):
    """Values between two codes go to the even one; a NaN or an infinity makes the head's scale
    NaN; subnormal heads and the largest singles keep their codes within 127."""
    hd, heads, kvh, rows = 64, 1, 1, 7
    x = np.zeros((rows, 3 * hd), np.float32)
    v = x[:, 2 * hd:]
    k = np.arange(hd - 1) * 4 - 125
    v[0, 0], v[0, 1:] = 127 * 0.375, (k + 0.5) * 0.375  # ties of both signs
    v[1] = 2.0
    v[1, 9] = np.nan
    v[2] = -1.0
    v[2, 63] = -np.inf
    v[3] = np.float32(1e-44) * (np.arange(hd) % 5)  # subnormal, and a scale of zero
    v[4] = np.finfo(np.float32).max * np.linspace(-1, 1, hd)
    v[5] = np.float32(2.0 ** -149) * 140 * np.linspace(-1, 1, hd)
    x[6, hd:2 * hd] = np.inf  # of k, with a value head of zeros
    bufs = [dev.out(rows * hd), dev.out(rows * hd), dev.out(rows * 4), dev.out(rows * 4)]
    pool = q8_pool([b.ptr for b in bufs], rows, 1, kvh, hd)
    q = dev(x)
    H.check(H.lib().ihip_enqueue_paged_qkrope(
        ctx.h, q, 3 * hd, q + 4 * hd, 3 * hd, q + 8 * hd, 3 * hd, rows, heads, 0, 0, 0.0, None,
        dev(np.zeros(rows, np.int32)), dev(np.arange(rows, dtype=np.int32)), C.byref(pool), 0), "store")
    codes = bufs[1].download(np.int8, rows * hd).reshape(rows, hd)
    sc = bufs[3].download(np.float32, rows)
    assert sc[0] == np.float32(0.375) and codes[0, 0] == 127
    assert np.array_equal(codes[0, 1:], np.rint(k + 0.5))
    assert np.isnan(sc[1:3]).all() and (codes[1:3] == 0).all()
    assert sc[3] == 0 and (codes[3] == 0).all()
    assert codes[4].max() == 127 and codes[4].min() == -127 and np.isfinite(sc[4])
    # 140 steps of 2^-149 over 127 are 1.1 of them: a scale of one, codes cut at 127
    assert sc[5] == np.float32(2.0 ** -149) and codes[5].max() == 127 and codes[5].min() == -127
    assert np.isnan(bufs[2].download(np.float32, rows)[6]) and sc[6] == 0


# ---------------------------------------------------------------------- read
@pytest.mark.parametrize("cache", ["q8", "f16", "bf16", "f32"])
@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("hd,kvh,ps,layout,lengths,first", [
    (128, 4, 16, "tokens", [0, 1, 16, 17, 0, 300, 33], None), (80, 3, 7, "heads", [5, 0, 0, 61, 8], [2, 0, 9, 1, 30]),
    (16, 1, 1, "tokens", [1], None), (512, 2, 64, "heads", [130, 1, 64, 2000], [0, 63, 64, 1]),
    (64, 8, 100, "tokens", [7000] * 3 + [0] * 300 + [1] * 70, None)])
def test_read(ctx, dev, cache, out, hd, kvh, ps, layout, lengths, first):
    rng = np.random.default_rng(hd + ps + len(lengths))
    n = len(lengths)
    start = np.array(first or [0] * n, np.int32)
    lengths = np.array(lengths, np.int32)
    width = max(1, int((-(-(start + lengths) // ps)).max()))
    pages = 40
    table = rng.integers(0, pages, (n, width)).astype(np.int32)
    table[0, 0] = pages  # outside the pool
    if n > 3:
        table[3, -1] = -1
    offsets = np.concatenate([[3], 3 + np.cumsum(lengths)]).astype(np.int32)
    rows = int(offsets[-1]) + 5
    shape = (pages, ps, kvh, hd)
    if cache == "q8":
        raw = [rng.integers(-128, 128, shape).astype(np.int8) for _ in range(2)]
        raw += [rng.standard_normal(shape[:3]).astype(np.float32) for _ in range(2)]
        # (exact in 64 bits: a value is rounded once, to the rows' type; to single and then to
        # half it would be off by half a step and 2^-13 of one)
        value = [raw[i].astype(np.float64) * raw[i + 2][..., None] for i in range(2)]
    else:
        raw = [R.pack(rng.standard_normal(shape), cache) for _ in range(2)]
        value = [R.unpack(a, cache) for a in raw]
    at = [dev(np.ascontiguousarray(a.transpose(order(layout)[:a.ndim]))) for a in raw]
    if cache == "q8":
        pool = q8_pool(at, pages, ps, kvh, hd, layout)
    else:
        st, _ = strides_of(layout, ps, kvh, hd)
        pool = H.Pages(k=at[0], v=at[1], pages=pages, page_stride=st[0], slot_stride=st[1], head_stride=st[2],
                       page_size=ps, kv_heads=kvh, head_dim=hd, dtype={"f16": H.F16, "bf16": H.BF16, "f32": H.F32}[cache])
    ot, dt = (H.F32, np.float32) if out == "f32" else (H.F16, np.float16)
    bufs = [dev.out(rows * kvh * hd * np.dtype(dt).itemsize) for _ in range(2)]
    H.check(H.lib().ihip_enqueue_paged_read(
        ctx.h, C.byref(pool), dev(table), width, dev(start) if first else 0, dev(offsets), n, rows, ot, bufs[0].ptr,
        bufs[1].ptr), "read")
    for b, val in zip(bufs, value):
        got = b.download(dt, rows * kvh * hd).reshape(rows, kvh, hd)
        want = np.zeros((rows, kvh, hd))
        for s in range(n):
            pos = start[s] + np.arange(lengths[s])
            page = table[s, pos // ps]
            ok = (page >= 0) & (page < pages)
            want[offsets[s]:offsets[s + 1]] = np.where(ok[:, None, None], val[page.clip(0, pages - 1), pos % ps], 0)
        inner = slice(offsets[0], offsets[-1])
        bad = got[inner] != want[inner].astype(dt)
        assert not bad.any(), (np.argwhere(bad)[:5].tolist(), got[inner][bad][:5], want[inner][bad][:5])
        assert (got[:3].view(np.uint8) == 0x5A).all() and (got[-5:].view(np.uint8) == 0x5A).all()


# ----------------------------------------------------------------- attention
class Batch:
    """Sequences over shuffled pages of codes; what no sequence holds has codes and NaN scales."""

    def __init__(self, rng, hd, heads, kvh, ps, lengths, width=None, spread=1.0):
        self.hd, self.heads, self.kvh, self.ps = hd, heads, kvh, ps
        self.lengths = np.array(lengths, np.int32)
        n = len(lengths)
        have = -(-self.lengths.clip(0) // ps)
        self.pages, self.width = int(have.sum()) + 3, width or max(1, int(have.max()) + 1)
        pick = rng.permutation(self.pages)
        self.table = rng.integers(-2 ** 31, 2 ** 31, (n, self.width)).astype(np.int32)
        held, at = np.zeros((self.pages, ps), bool), 0
        for s in range(n):
            m = min(int(have[s]), self.width)
            self.table[s, :m] = pick[at:at + m]
            at += int(have[s])
            for p, t in R.keys_of(self.table[s], self.lengths[s], 0, ps, self.pages):
                held[p, t] = True
        shape = (self.pages, ps, kvh, hd)
        self.codes = [rng.integers(-128, 128, shape).astype(np.int8) for _ in range(2)]
        # scales of any size and sign
        self.scales = [(np.exp(spread * rng.standard_normal(shape[:3])) / 73 * rng.choice([1, 1, 1, -1], shape[:3]))
                       .astype(np.float32) for _ in range(2)]
        for sc in self.scales:
            sc[~held] = np.nan
        self.q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        self.sinks, self.window, self.scale, self.layout, self.pad = None, 0, 0.0, "tokens", 0

    def upload(self, dev):
        o = order(self.layout)
        at = [dev(np.ascontiguousarray(a.transpose(o[:a.ndim]))) for a in self.codes + self.scales]
        self.pool = q8_pool(at, self.pages, self.ps, self.kvh, self.hd, self.layout)
        n = len(self.q)
        rows = np.full((n, self.heads * self.hd + self.pad), np.nan, np.float32)
        rows[:, :self.heads * self.hd] = self.q.reshape(n, -1)
        self.dq, self.dt, self.dl = dev(rows), dev(self.table), dev(self.lengths)
        self.ds = dev(self.sinks) if self.sinks is not None else 0
        self.y = dev.out(self.q.nbytes)

    def enqueue(self, ctx):
        H.check(H.lib().ihip_enqueue_paged_attention(
            ctx.h, self.dq, self.heads * self.hd + self.pad if self.pad else 0, C.byref(self.pool), self.dt,
            self.width, self.dl, self.y.ptr, len(self.lengths), self.heads, self.window, self.ds, self.scale), "attention")

    def read(self):
        return self.y.download(np.float32, self.q.size).reshape(self.q.shape)

    def want(self):
        """The definition, and what sums in single may be off by (paged_ref.attention). A query
        is two halves: 2^-23 of it and so 2 U more of a score's magnitudes. A weight times its
        scale is two halves below the largest scale: 2^-22 of it, and 2^-39 of that scale for a
        small one."""
        k, v = (c.astype(np.float64) * s[..., None].astype(np.float64) for c, s in zip(self.codes, self.scales))
        with np.errstate(invalid="ignore", over="ignore"):
            y, tol = R.attention(self.q.astype(np.float64), k, v, self.table, self.lengths, self.ps, self.window,
                                 self.sinks, self.scale)
        for s in range(len(self.q)):
            at = R.keys_of(self.table[s], self.lengths[s], self.window, self.ps, self.pages)
            if at:
                big = np.abs(np.array([self.scales[1][p, t] for p, t in at])).max(0) * 128  # of each KV head
                tol[s] += 2.0 ** -39 * len(at) * np.repeat(big, self.heads // self.kvh)[:, None]
        return y, tol

    def check(self, ctx, dev):
        self.upload(dev)
        self.enqueue(ctx)
        got, (want, tol), live = self.read(), self.want(), self.lengths >= 0
        assert (got[~live].view(np.uint8) == 0x5A).all()
        assert_close(got[live], want[live], tol[live])
        return got


SHAPES = [(128, 32, 4, 16), (64, 64, 8, 32), (256, 8, 2, 64), (512, 16, 2, 16), (96, 12, 12, 7), (80, 32, 2, 1),
          (16, 3, 1, 24), (128, 48, 2, 256), (144, 17, 1, 100), (512, 2, 2, 1), (272, 4, 4, 8)]


@pytest.mark.parametrize("hd,heads,kvh,ps", SHAPES)
def test_attention(ctx, dev, hd, heads, kvh, ps):
    Batch(np.random.default_rng(hd + heads + ps), hd, heads, kvh, ps, LENGTHS).check(ctx, dev)


@pytest.mark.parametrize("window,sinks,scale,layout,pad,spread", [
    (1, False, 0.0, "tokens", 0, 1.0), (16, True, 0.0, "heads", 8, 0.0), (33, False, 0.3, "tokens", 3, 2.0),
    (128, True, 0.0, "tokens", 0, 1.0), (10 ** 6, True, 0.05, "heads", 0, 1.0), (0, True, 0.5, "heads", 64, 0.5)])
def test_attention_windows_sinks_strides(ctx, dev, window, sinks, scale, layout, pad, spread):
    rng = np.random.default_rng(window + pad)
    b = Batch(rng, 64, 8, 2, 16, LENGTHS + [300, 700], spread=spread)
    b.window, b.scale, b.layout, b.pad = window, scale, layout, pad
    b.sinks = (rng.standard_normal(8) * 2).astype(np.float32) if sinks else None
    b.check(ctx, dev)


@pytest.mark.parametrize("hd,heads,kvh,ps,lengths", [
    (128, 8, 2, 16, [30000]), (64, 8, 1, 32, [9000, 3, 12000]), (256, 4, 1, 64, [5000, 20000]),
    (512, 4, 1, 16, [6000]), (64, 64, 64, 64, [8300, 0, 8400])])
def test_attention_split_over_the_length(ctx, dev, hd, heads, kvh, ps, lengths):
    Batch(np.random.default_rng(hd), hd, heads, kvh, ps, lengths).check(ctx, dev)


def test_attention_scales_that_grow(ctx, dev):
    """The largest value scale of a wave's keys rises step by step, falls, and starts at zero."""
    rng = np.random.default_rng(4)
    b = Batch(rng, 128, 8, 2, 16, [700, 500, 260])
    for s, sizes in enumerate((np.linspace(-9, 9, 700), np.linspace(4, -20, 500), np.full(260, -200.0))):
        for j, e in enumerate(sizes):
            b.scales[1][b.table[s, j // 16], j % 16] = np.ldexp(1.0, int(np.round(e))) if e > -100 else 0.0
    got = b.check(ctx, dev)
    assert (got[2] == 0).all()


def test_attention_pages_that_are_not_there(ctx, dev):
    rng = np.random.default_rng(6)
    b = Batch(rng, 128, 8, 2, 16, [100, 60, 30, 33])
    b.table[0, 2], b.table[1, :], b.table[3, 2] = -1, b.pages, -2 ** 31
    b.sinks = rng.standard_normal(8).astype(np.float32)
    assert (b.check(ctx, dev)[1] == 0).all()


def test_attention_infinities_and_nan(ctx, dev):
    """A scale of NaN is a head of NaN, an infinite one infinities and NaN: in their own
    sequence and KV head alone."""
    rng = np.random.default_rng(8)
    b = Batch(rng, 128, 8, 2, 16, [50, 50, 200, 40, 64])
    b.scales[0][b.table[0, 1], 3, 0] = np.nan
    b.scales[1][b.table[1, 0], 5, 1] = np.nan
    b.codes[1][b.table[2, 9], 2, 0] = np.abs(b.codes[1][b.table[2, 9], 2, 0].astype(int)).clip(1, 127)
    b.scales[1][b.table[2, 9], 2, 0] = np.inf
    b.q[3, 2, 7] = np.nan
    b.upload(dev)
    b.enqueue(ctx)
    got, (want, tol) = b.read(), b.want()
    assert np.isnan(got[0, :4]).all() and np.isnan(got[1, 4:]).all() and np.isnan(got[3, 2]).all()
    assert (got[2, :4] == np.inf).all()
    ok = np.ones(got.shape[:2], bool)
    ok[0, :4] = ok[1, 4:] = ok[2, :4] = ok[3, 2] = False
    assert_close(got[ok], want[ok], tol[ok])


def test_past_32_bits(ctx, dev):
    """Keys whose codes lie more than 2^31 values into the pool, in pages that lie apart."""
    rng = np.random.default_rng(9)
    hd, heads, kvh, ps, pages = 128, 4, 1, 16, 3
    stride = (1 << 31) + 128 * 16 * 5
    n = stride * (pages - 1) + ps * hd
    k = [ctx.alloc(n) for _ in range(2)]
    s = [ctx.alloc(n // hd * 4 + 4) for _ in range(2)]
    try:
        codes = [rng.integers(-127, 128, (pages, ps, kvh, hd)).astype(np.int8) for _ in range(2)]
        scales = [rng.random((pages, ps, kvh)).astype(np.float32) / 100 for _ in range(2)]
        for i in range(2):
            for p in range(pages):
                a, c = codes[i][p].copy(), scales[i][p].copy()
                H.check(H.lib().ihip_upload(ctx.h, k[i].ptr + p * stride, a.ctypes.data, a.nbytes))
                H.check(H.lib().ihip_upload(ctx.h, s[i].ptr + p * stride // hd * 4, c.ctypes.data, c.nbytes))
        pool = H.Pages(k=k[0].ptr, v=k[1].ptr, pages=pages, page_stride=stride, page_size=ps, kv_heads=kvh, head_dim=hd,
                       dtype=H.Q8_HEAD, k_scale=s[0].ptr, v_scale=s[1].ptr)
        table, lengths = np.array([[2, 0, 1]], np.int32), np.array([45], np.int32)
        q = rng.standard_normal((1, heads, hd)).astype(np.float32)
        y, rows = dev.out(q.nbytes), [dev.out(45 * hd * 4) for _ in range(2)]
        H.check(H.lib().ihip_enqueue_paged_attention(ctx.h, dev(q), 0, C.byref(pool), dev(table), 3, dev(lengths),
                                                     y.ptr, 1, heads, 0, 0, 0.0))
        H.check(H.lib().ihip_enqueue_paged_read(ctx.h, C.byref(pool), dev(table), 3, 0, dev(np.array([0, 45], np.int32)),
                                                1, 45, H.F32, rows[0].ptr, rows[1].ptr))
        val = [c.astype(np.float32) * x[..., None] for c, x in zip(codes, scales)]
        want, tol = R.attention(q.astype(np.float64), *(v.astype(np.float64) for v in val), table, lengths, ps)
        assert_close(y.download(np.float32, q.size).reshape(q.shape), want, tol + 2.0 ** -39 * 45 * 1.3)
        for b, v in zip(rows, val):
            assert np.array_equal(b.download(np.float32, 45 * hd), v[[2, 0, 1]].reshape(-1)[:45 * hd])
    finally:
        ctx.sync()
        for b in k + s:
            b.free()


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("graph", [False, True])
def test_steps_together(ctx, dev, graph):
    """Prompts stored into 8-bit pages, then decode steps: plan, store, attention, and the whole
    histories read back, which are what the attention used."""
    hd, heads, kvh, ps, width, n, pages = 64, 8, 2, 4, 16, 4, 40
    rng = np.random.default_rng(22)
    past, prompt = np.zeros(n, np.int32), np.array([9, 1, 30, 17], np.int32)
    table, ring = np.full((n, width), -1, np.int32), rng.permutation(pages).astype(np.int32)
    freq = (1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd)).astype(np.float32)
    rope, cap, row = H.Rope(freq=dev(freq)), 64, (heads + 2 * kvh) * hd
    b = {}
    for name, a in dict(past=past, table=table, ring=ring, ends=np.array([0, pages], np.int64)).items():
        b[name] = dev.out(a.nbytes)
        b[name].upload(a)
    bufs = [dev.out(pages * ps * kvh * hd) for _ in range(2)] + [dev.out(pages * ps * kvh * 4, 0xFF) for _ in range(2)]
    pool = q8_pool([x.ptr for x in bufs], pages, ps, kvh, hd)
    dcount, dx, y = dev.out(4 * n), dev.out(cap * row * 4), dev.out(n * heads * hd * 4)
    offs, pos, slots, failed = dev.out(4 * n + 4), dev.out(4 * cap), dev.out(4 * cap), dev.out(4)
    bound = width * ps * n
    every = dev(np.arange(0, bound + 1, width * ps, dtype=np.int32))  # rows for full tables
    back = [dev.out(bound * kvh * hd * 4) for _ in range(2)]
    L = H.lib()

    def step(rows):
        H.check(L.ihip_enqueue_paged_slots(
            ctx.h, b["past"].ptr, dcount.ptr, n, b["table"].ptr, width, ps, b["ring"].ptr, pages, b["ends"].ptr,
            b["ends"].ptr, offs.ptr, b["past"].ptr, pos.ptr, slots.ptr, rows, failed.ptr))
        q = dx.ptr
        H.check(L.ihip_enqueue_paged_qkrope(
            ctx.h, q, row, q + 4 * heads * hd, row, q + 4 * (heads + kvh) * hd, row, rows, heads, 0, 0, 0.0,
            C.byref(rope), pos.ptr, slots.ptr, C.byref(pool), 0))

    def rest():
        H.check(L.ihip_enqueue_paged_attention(ctx.h, dx.ptr, row, C.byref(pool), b["table"].ptr, width, b["past"].ptr,
                                               y.ptr, n, heads, 0, 0, 0.0))
        H.check(L.ihip_enqueue_paged_read(ctx.h, C.byref(pool), b["table"].ptr, width, 0, every, n, bound, H.F32,
                                          back[0].ptr, back[1].ptr))

    dcount.upload(prompt)
    dx.upload(rng.standard_normal((cap, row)).astype(np.float32))
    step(cap)
    dcount.upload(np.ones(n, np.int32))
    if graph:
        H.check(L.ihip_capture_begin(ctx.h))
        step(n), rest()
        H.check(L.ihip_capture_end(ctx.h, 11))
    lengths = prompt.copy()
    for _ in range(5):
        dx.upload(rng.standard_normal((n, row)).astype(np.float32))
        if graph:
            H.check(L.ihip_graph_launch(ctx.h, 11))
        else:
            step(n), rest()
        lengths = lengths + 1
        assert np.array_equal(b["past"].download(np.int32, n), lengths) and failed.download(np.int32, 1)[0] == 0
        t = b["table"].download(np.int32, n * width).reshape(n, width)
        k, v = (x.download(np.float32, bound * kvh * hd).reshape(n, width * ps, kvh, hd) for x in back)
        q = dx.download(np.float32, n * row).reshape(n, row)[:, :heads * hd].reshape(n, heads, hd).astype(np.float64)
        # the histories as one pool: sequence s's are pages s * width ..
        kk, vv = (a.reshape(n * width, ps, kvh, hd).astype(np.float64) for a in (k, v))
        mine = np.arange(n * width).reshape(n, width).astype(np.int32)
        want, tol = R.attention(q, kk, vv, mine, lengths, ps)
        # (the values read back are products rounded to single, which the attention's are not)
        top_k, top_v = (max(np.abs(a[s, :lengths[s]]).max() for s in range(n)) for a in (k, v))
        room = 4 * U * (top_v + top_k * np.abs(q).max() * hd * top_v) + 2.0 ** -39 * 64 * top_v
        assert_close(y.download(np.float32, q.size).reshape(q.shape), want, tol + room)
        assert all((t[s, :-(-lengths[s] // ps)] >= 0).all() for s in range(n))
        for s in range(n):  # tokens in pages that are not taken yet read as zeros
            assert (k[s, -(-lengths[s] // ps) * ps:] == 0).all()

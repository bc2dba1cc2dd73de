"""Attention of groups that share their first tokens, on the device, against the
attention of every sequence over its own table in 64 bits (paged_ref.py)."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_ref as R
from test_gpu_paged import assert_close, ctx, dev, pages_struct, strides_of  # noqa: F401 (fixtures)
from test_gpu_paged_q8 import order, q8_pool

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16", "q8"]


class Batch:
    """Groups of sequences [(members, shared tokens, tokens that every member's table really has in
    common)] behind `alone` sequences of no group, lengths by sequence."""

    def __init__(self, rng, dtype, hd, heads, kvh, ps, groups, lengths, alone=0, behind=0):
        self.dtype, self.hd, self.heads, self.kvh, self.ps = dtype, hd, heads, kvh, ps
        n = alone + sum(g[0] for g in groups) + behind
        self.lengths = np.resize(np.array(lengths, np.int32), n)
        self.members = np.cumsum([alone] + [g[0] for g in groups]).astype(np.int32)
        self.shared = np.array([g[1] for g in groups], np.int32)
        have = -(-self.lengths.clip(0) // ps)
        common = [-(-g[2] // ps) for g in groups]
        self.width = max([1, int(have.max())] + common) + 1
        self.pages = int(have.sum()) + sum(common) + 3
        pick, at = rng.permutation(self.pages), 0
        self.table = rng.integers(-2 ** 31, 2 ** 31, (n, self.width)).astype(np.int32)
        for s in range(n):
            self.table[s, :have[s]] = pick[at:at + have[s]]
            at += have[s]
        for g, m in enumerate(common):
            self.table[self.members[g]:self.members[g + 1], :m] = pick[at:at + m]
            at += m
        shape = (self.pages, ps, kvh, hd)
        if dtype == "q8":
            self.raw = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            self.raw += [(np.exp(0.5 * rng.standard_normal(shape[:3])) / 73).astype(np.float32) for _ in range(2)]
        else:
            self.raw = [R.pack(rng.standard_normal(shape), dtype) for _ in range(2)]
        # tokens that no sequence holds and no prefix has: NaN
        held = np.zeros((self.pages, ps), bool)
        for s in range(n):
            for p, t in R.keys_of(self.table[s], self.lengths[s], 0, ps, self.pages):
                held[p, t] = True
        for g in range(len(groups)):
            for p, t in R.keys_of(self.table[self.members[g]], self.shared[g], 0, ps, self.pages):
                held[p, t] = True
        for a in self.raw[2:] if dtype == "q8" else self.raw:
            a[~held] = R.pack(np.array([np.nan]), dtype)[0] if dtype == "bf16" else np.nan
        self.q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        self.sinks, self.window, self.scale, self.layout, self.pad, self.offsets = None, 0, 0.0, "tokens", 0, None

    def values(self):
        if self.dtype == "q8":
            return [c.astype(np.float64) * s[..., None] for c, s in zip(self.raw[:2], self.raw[2:])]
        return [R.unpack(a, self.dtype) for a in self.raw]

    def upload(self, dev):
        o, n = order(self.layout), len(self.q)
        at = [dev(np.ascontiguousarray(a.transpose(o[:a.ndim]))) for a in self.raw]
        self.pool = q8_pool(at, self.pages, self.ps, self.kvh, self.hd, self.layout) if self.dtype == "q8" else \
            pages_struct(at[0], at[1], self.pages, self.ps, self.kvh, self.hd, self.dtype, self.layout)
        self.rows = n if self.offsets is None else int(self.offsets[-1])
        self.row = np.arange(n) if self.offsets is None else self.offsets[1:] - 1
        x = np.full((self.rows, self.heads * self.hd + self.pad), np.nan, np.float32)
        x[self.row, :self.heads * self.hd] = self.q.reshape(n, -1)
        self.dq, self.dt, self.dl = dev(x), dev(self.table), dev(self.lengths)
        self.dm, self.dsh = dev(self.members), dev(self.shared)
        self.ds = dev(self.sinks) if self.sinks is not None else 0
        self.do = dev(self.offsets) if self.offsets is not None else 0
        self.y = dev.out(self.rows * self.heads * self.hd * 4)

    def enqueue(self, ctx):
        H.check(H.lib().ihip_enqueue_paged_attention_shared(
            ctx.h, self.dq, self.heads * self.hd + self.pad if self.pad else 0, C.byref(self.pool), self.dt, self.width,
            self.dl, self.do, self.rows, self.dm, self.dsh, len(self.shared), self.y.ptr, len(self.q), self.heads,
            self.window, self.ds, self.scale), "shared")

    def read(self):
        return self.y.download(np.float32, self.rows * self.heads * self.hd).reshape(self.rows, self.heads, self.hd)

    def want(self):
        """paged_ref.attention's bound holds for sums in any order; 8-bit pages' small weights are
        off by 2^-39 of the largest scale more (test_gpu_paged_q8.py), here of the prefix and
        the own tokens each."""
        with np.errstate(invalid="ignore", over="ignore"):
            y, tol = R.attention(self.q.astype(np.float64), *self.values(), self.table, self.lengths, self.ps, self.window,
                                 self.sinks, self.scale)
        if self.dtype == "q8":
            for s in range(len(self.q)):
                at = R.keys_of(self.table[s], self.lengths[s], self.window, self.ps, self.pages)
                if at:
                    big = np.abs(np.array([self.raw[3][p, t] for p, t in at])).max(0) * 128
                    tol[s] += 2.0 ** -39 * len(at) * np.repeat(big, self.heads // self.kvh)[:, None]
        return y, tol

    def check(self, ctx, dev, twice=False):
        self.upload(dev)
        self.enqueue(ctx)
        got, (want, tol) = self.read(), self.want()
        live = self.lengths >= 0
        rest = np.ones(self.rows, bool)
        rest[self.row[live]] = False
        assert (got[rest].view(np.uint8) == 0x5A).all()
        assert_close(got[self.row[live]], want[live], tol[live])
        return got[self.row]


SHAPES = [(128, 32, 4, 16), (64, 64, 8, 32), (256, 8, 2, 64), (512, 16, 2, 16), (96, 12, 12, 7), (80, 32, 2, 1),
          (16, 3, 1, 24), (128, 48, 2, 256), (144, 17, 1, 100), (512, 2, 2, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,kvh,ps", SHAPES)
def test_groups(ctx, dev, dtype, hd, heads, kvh, ps):
    """Groups of one to many, some sequences before and behind them, prefixes of part of a page's
    tokens, of one token, of nothing."""
    rng = np.random.default_rng(hd + heads + ps)
    b = Batch(rng, dtype, hd, heads, kvh, ps, [(2, 130, 130), (1, 40, 64), (9, 257, 300), (3, 1, 1), (4, 0, 33), (2, 64, 64)],
              [300, 301, 310, 333, 420, 305, 299, 300], alone=1, behind=2)
    b.check(ctx, dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sinks,scale,layout,pad,window", [(True, 0.0, "heads", 8, 0), (False, 0.4, "tokens", 3, 0),
                                                           (True, 0.1, "tokens", 0, 90), (True, 0.0, "tokens", 0, 0)])
def test_short_sequences_sinks_strides(ctx, dev, dtype, sinks, scale, layout, pad, window):
    """Members shorter than the prefix, without a token, ended ones; every length beside its end."""
    rng = np.random.default_rng(pad + window)
    b = Batch(rng, dtype, 64, 8, 2, 16, [(30, 200, 200), (5, 16, 16)],
              [200, 0, -1, 1, 199, 201, 16, 15, 17, 31, 32, 33, 128, 129, 127, 250, -1, 330, 64, 260, 0], alone=2)
    b.sinks = (rng.standard_normal(8) * 2).astype(np.float32) if sinks else None
    b.scale, b.layout, b.pad, b.window = scale, layout, pad, window
    b.check(ctx, dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,kvh,groups,own", [
    (128, 4, 2, [(2, 20000, 20000)], 5), (64, 64, 8, [(20, 3000, 3000)], 700), (256, 4, 1, [(3, 9000, 9000), (2, 500, 500)], 1500),
    (512, 4, 2, [(3, 2500, 2500)], 60), (128, 24, 2, [(7, 1100, 1100)] * 3, 0)])
def test_prefixes_that_blocks_share(ctx, dev, dtype, hd, heads, kvh, groups, own):
    rng = np.random.default_rng(hd + own)
    lengths = [g[1] + int(rng.integers(0, own + 1)) for g in groups for _ in range(g[0])]
    Batch(rng, dtype, hd, heads, kvh, 32, groups, lengths).check(ctx, dev)


@pytest.mark.parametrize("dtype", ["f16", "q8"])
def test_many_groups(ctx, dev, dtype):
    """More groups than lanes, of a few tiles each: whole prefixes to a block, and several."""
    rng = np.random.default_rng(3)
    groups = [(2 + i % 3, 30 + 17 * i % 400, 30 + 17 * i % 400) for i in range(150)]
    lengths = [g[1] + 1 + j for g in groups for j in range(g[0])]
    Batch(rng, dtype, 64, 8, 2, 16, groups, lengths, alone=3, behind=1).check(ctx, dev)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_a_step(ctx, dev, dtype):
    """Sequences' last rows of a step with several rows each; rows that no sequence ends are left."""
    rng = np.random.default_rng(5)
    b = Batch(rng, dtype, 128, 16, 8, 16, [(5, 90, 96), (3, 40, 48)], [100, 95, 140, 97, 300, 60, 41, 50])
    b.offsets = np.cumsum([0, 3, 1, 2, 1, 1, 4, 1, 2]).astype(np.int32)
    b.check(ctx, dev)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_not_there_infinities_and_nan(ctx, dev, dtype):
    rng = np.random.default_rng(7)
    b = Batch(rng, dtype, 128, 8, 2, 16, [(4, 160, 160), (3, 100, 112), (3, 64, 64)], [200, 161, 180, 100, 130, 101, 300, 90, 70, 65])
    b.table[0:4, 3] = -1
    b.table[4:7, :7] = b.pages  # the second group's prefix is gone
    p = b.table[7, 1]
    if dtype == "q8":
        b.raw[3][p, 5, 1] = np.nan
    elif dtype == "bf16":
        b.raw[1][p, 5, 1, 9] = 0x7FC0
    else:
        b.raw[1][p, 5, 1, 9] = np.nan
    b.q[1, 6, 3] = np.nan
    b.sinks = rng.standard_normal(8).astype(np.float32)
    b.upload(dev)
    b.enqueue(ctx)
    got, (want, tol) = b.read(), b.want()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan) and nan[1, 6].all() and nan[7:, 4:].any() and not nan[7:, :4].any()
    ok = ~nan.any(-1)
    assert_close(got[ok], want[ok], tol[ok])
    single = ok.copy()
    single[:] = False
    single[7:, 4:] = True  # (a NaN of one value is in that dimension alone)
    single &= dtype != "q8"
    if single.any():
        keep = ~nan & single[..., None]
        bad = ~(np.abs(got - want) <= tol) & keep
        assert not (bad & ~np.isnan(tol)).any()


def test_the_same_as_without_groups(ctx, dev):
    """No prefix at all, or none of two: bit by bit the attention without groups."""
    rng = np.random.default_rng(9)
    b = Batch(rng, "bf16", 128, 16, 4, 16, [(1, 50, 50), (3, 0, 0), (1, 64, 64)], [1500, 3, 700, 64, 65])
    b.sinks = rng.standard_normal(16).astype(np.float32)
    got = b.check(ctx, dev)
    y = dev.out(b.q.nbytes)
    H.check(H.lib().ihip_enqueue_paged_attention(ctx.h, b.dq, 0, C.byref(b.pool), b.dt, b.width, b.dl, y.ptr, len(b.q), 16,
                                                 0, b.ds, 0.0))
    assert np.array_equal(y.download(np.uint32, b.q.size), got.view(np.uint32).ravel())


def test_arrays_out_of_order(ctx, dev):
    """Members that do not ascend, lie outside the batch or overlap, and lengths of prefixes of any
    size: the call ends, and what lies behind the rows is left."""
    rng = np.random.default_rng(11)
    for members, shared in (([5, 2, 9, 0], [64, 64, 64]), ([-3, 4, 100, 2 ** 31 - 1], [10 ** 9, -5, 2 ** 31 - 1]),
                            ([0, 8, 0, 8], [100, 100, 100]), ([3, 3, 3, 3], [9, 9, 9])):
        b = Batch(rng, "f16", 64, 8, 2, 16, [(8, 64, 64)], [100, 80, 70, 90, 64, 130, 65, 99])
        b.members, b.shared = np.array(members, np.int32), np.array(shared, np.int32)
        b.upload(dev)
        tail = dev.out(b.q.nbytes + 4096)
        b.y = tail
        b.enqueue(ctx)
        assert (tail.download(np.uint8, b.q.nbytes + 4096)[b.q.nbytes:] == 0x5A).all()


def test_captured_and_replayed(ctx, dev):
    """Two graphs of one context over its workspaces, replayed in turn as lengths and groups
    change, with eager calls between; results do not change from run to run."""
    rng = np.random.default_rng(13)
    bs = [Batch(rng, "bf16", 64, 16, 2, 16, [(6, 400, 400), (4, 90, 96)], [450] * 10),
          Batch(rng, "q8", 128, 8, 4, 32, [(7, 1000, 1024), (3, 64, 64)], [1100] * 10)]
    bufs = []
    for i, b in enumerate(bs):
        b.upload(dev)
        bufs.append({k: dev.out(a.nbytes) for k, a in (("dl", b.lengths), ("dm", b.members), ("dsh", b.shared))})
        for k, v in bufs[i].items():
            setattr(b, k, v.ptr)
        H.check(H.lib().ihip_capture_begin(ctx.h))
        b.enqueue(ctx)
        H.check(H.lib().ihip_capture_end(ctx.h, 12 + i))
    for step in range(5):
        for i, b in enumerate(bs):
            most = int(b.shared[0])
            b.lengths = rng.integers(1, most + 40, 10).astype(np.int32)
            cut = int(rng.integers(0, 11))
            b.members = np.array([0, cut, 10 if step % 2 else cut], np.int32)
            # what both parts of the batch have in common in this table
            first = [64 if most < 500 else 32, 0]
            b.shared = np.array([most if cut <= (6 if i == 0 else 7) else 0, first[1]], np.int32)
            b.lengths[cut:] = b.lengths[cut:].clip(1, 400)
            for k, a in (("dl", b.lengths), ("dm", b.members), ("dsh", b.shared)):
                bufs[i][k].upload(a)
            H.check(H.lib().ihip_graph_launch(ctx.h, 12 + i))
        outs = [b.read() for b in bs]
        for b, got in zip(bs, outs):
            b.y.upload(np.full(got.nbytes, 0x5A, np.uint8))
            b.enqueue(ctx)
            assert np.array_equal(b.read().view(np.uint32), got.view(np.uint32))
            with np.errstate(invalid="ignore"):
                want, tol = b.want()
            ok = np.isfinite(tol).all((1, 2))
            assert ok.sum() >= 5
            assert_close(got[ok], want[ok], tol[ok])


@pytest.mark.parametrize("dtype", ["f16", "q8"])
def test_past_32_bits(ctx, dev, dtype):
    """A prefix and own tokens more than 2^31 values into the pool, in pages that lie apart."""
    rng = np.random.default_rng(15)
    hd, heads, kvh, ps, pages = 128, 4, 1, 16, 4
    stride, es = (1 << 30) + 128 * 16 * 5, 1 if dtype == "q8" else 2
    n = stride * (pages - 1) + ps * hd
    shape, values = (pages, ps, kvh, hd), []
    held = [ctx.alloc(n * es) for _ in range(2)] + ([ctx.alloc(n // hd * 4 + 4) for _ in range(2)] if dtype == "q8" else [])
    try:
        if dtype == "q8":
            raw = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            raw += [(rng.random(shape[:3]) / 73).astype(np.float32) for _ in range(2)]
            values = [c.astype(np.float64) * s[..., None] for c, s in zip(raw[:2], raw[2:])]
        else:
            raw = [R.pack(rng.standard_normal(shape), dtype) for _ in range(2)]
            values = [R.unpack(a, dtype) for a in raw]
        for i, a in enumerate(raw):
            for p in range(pages):
                page = np.ascontiguousarray(a[p])
                step = stride * es if i < 2 else stride // hd * 4
                H.check(H.lib().ihip_upload(ctx.h, held[i].ptr + p * step, page.ctypes.data, page.nbytes))
        pool = H.Pages(k=held[0].ptr, v=held[1].ptr, pages=pages, page_stride=stride, page_size=ps, kv_heads=kvh, head_dim=hd,
                       dtype=H.Q8_HEAD if dtype == "q8" else H.F16, k_scale=held[2].ptr if dtype == "q8" else 0,
                       v_scale=held[3].ptr if dtype == "q8" else 0)
        table, lengths = np.array([[3, 1, 0], [3, 1, 2]], np.int32), np.array([45, 41], np.int32)
        q = rng.standard_normal((2, heads, hd)).astype(np.float32)
        y = dev.out(q.nbytes)
        H.check(H.lib().ihip_enqueue_paged_attention_shared(
            ctx.h, dev(q), 0, C.byref(pool), dev(table), 3, dev(lengths), 0, 2, dev(np.array([0, 2], np.int32)),
            dev(np.array([30], np.int32)), 1, y.ptr, 2, heads, 0, 0, 0.0))
        want, tol = R.attention(q.astype(np.float64), *values, table, lengths, ps)
        # (8-bit pages' small weights are off by 2^-39 of the largest scale more)
        assert_close(y.download(np.float32, q.size).reshape(q.shape), want,
                     tol + (2.0 ** -39 * 45 * 128 / 73 if dtype == "q8" else 0))
    finally:
        ctx.sync()
        for b in held:
            b.free()

"""The paged operators on the host (no device): refused calls, the index
arithmetic of lengths, pages and slots at its borders, the oracle's plan, and
the rotary frequencies."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import oracle_lib as O
import paged_ref as R
from infer_hip import models

A = 1 << 20  # an address that no check follows


def refused(call, rc, text):
    got = call()
    assert got == rc, (got, H.lib().ihip_last_error())
    assert text in H.lib().ihip_last_error().decode(), H.lib().ihip_last_error()


def pages(**kw):
    a = dict(k=A, v=A, pages=8, page_size=16, kv_heads=2, head_dim=64, dtype=H.F16)
    a.update(kw)
    return H.Pages(**a)


BAD_POOLS = [
    (dict(k=0), -1, "no cache"), (dict(v=0), -1, "no cache"), (dict(k=A + 8), -1, "aligned"),
    (dict(dtype=H.Q8_0), -3, "F32, F16 or BF16"), (dict(dtype=0), -3, "F32, F16 or BF16"),
    (dict(head_dim=0), -3, "head_dim"), (dict(head_dim=60), -3, "head_dim"),
    (dict(head_dim=520), -3, "head_dim"), (dict(kv_heads=0), -1, "out of range"),
    (dict(page_size=0), -1, "out of range"), (dict(page_size=-16), -1, "out of range"),
    (dict(pages=0), -1, "out of range"), (dict(pages=1 << 27), -1, "out of range"),
    (dict(pages=1 << 62), -1, "out of range"),
    (dict(slot_stride=63), -1, "stride"), (dict(head_stride=-64), -1, "stride"),
    (dict(slot_stride=132), -1, "stride"), (dict(page_stride=32), -1, "stride"),
    (dict(page_stride=1 << 41), -1, "stride"), (dict(slot_stride=1 << 30), -1, "page of more"),
]


def attention(pool, **kw):
    a = dict(ctx=None, q=A, q_stride=0, table=A, max_pages=4, lengths=A, y=A, seqs=3, heads=4,
             window=0, sinks=0, scale=0.0)
    a.update(kw)
    p = C.byref(pool) if pool is not None else None
    return H.lib().ihip_enqueue_paged_attention(
        a["ctx"], a["q"], a["q_stride"], p, a["table"], a["max_pages"], a["lengths"], a["y"],
        a["seqs"], a["heads"], a["window"], a["sinks"], a["scale"])


def qkrope(pool, rope=None, **kw):
    a = dict(q=A, qs=0, k=A, ks=0, v=A, vs=0, rows=5, heads=4, qn=0, kn=0, eps=1e-6, positions=A,
             slots=A, out=0)
    a.update(kw)
    return H.lib().ihip_enqueue_paged_qkrope(
        None, a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["rows"], a["heads"], a["qn"],
        a["kn"], a["eps"], C.byref(rope) if rope is not None else None, a["positions"], a["slots"],
        C.byref(pool) if pool is not None else None, a["out"])


@pytest.mark.parametrize("bad,rc,text", BAD_POOLS)
def test_pools_refused(bad, rc, text):
    refused(lambda: attention(pages(**bad)), rc, text)
    refused(lambda: qkrope(pages(**bad)), rc, text)


def test_attention_refused():
    refused(lambda: attention(None), -1, "no cache")
    for name in ("q", "table", "lengths", "y"):
        refused(lambda: attention(pages(), **{name: 0}), -1, "missing array")
        refused(lambda: attention(pages(), **{name: A + 2}), -1, "aligned")
    for bad in (dict(seqs=0), dict(seqs=-1), dict(heads=0), dict(heads=3), dict(heads=65536),
                dict(window=-1), dict(max_pages=0), dict(max_pages=1 << 28)):
        refused(lambda: attention(pages(), **bad), -1, "out of range")
    refused(lambda: attention(pages(), seqs=H.PAGED_SEQS + 1), -6, "IHIP_PAGED_SEQS")
    refused(lambda: attention(pages(), q_stride=255), -1, "stride below")
    refused(lambda: attention(pages(), q_stride=1 << 37), -1, "2^36")
    # tables whose tiles of keys pass 32 bits
    refused(lambda: attention(pages(page_size=1 << 20, pages=2, kv_heads=2, head_dim=8), max_pages=1 << 10,
                              seqs=4096, heads=64), -6, "2^31 tiles")
    for bad in (float("nan"), float("inf")):
        refused(lambda: attention(pages(), scale=bad), -1, "scale")
    # everything in order but the context
    refused(lambda: attention(pages()), -1, "no context")
    refused(lambda: attention(pages(slot_stride=64, head_stride=1024)), -1, "no context")


def test_attention_at_refused():
    def call(**kw):
        a = dict(q=A, qs=0, pool=C.byref(pages()), table=A, mp=4, lengths=A, offsets=A, rows=5, y=A, seqs=3,
                 heads=4, window=0, sinks=0, scale=0.0)
        a.update(kw)
        return H.lib().ihip_enqueue_paged_attention_at(None, *a.values())

    for bad in (dict(rows=0), dict(rows=-1), dict(rows=1 << 31), dict(seqs=0)):
        refused(lambda: call(**bad), -1, "out of range")
    refused(lambda: call(offsets=A + 1), -1, "aligned")
    refused(lambda: call(lengths=0), -1, "missing array")
    refused(lambda: call(), -1, "no context")


def test_qkrope_refused():
    refused(lambda: qkrope(None), -1, "no cache")
    for name in ("q", "k", "v", "positions", "slots"):
        refused(lambda: qkrope(pages(), **{name: 0}), -1, "missing array")
    for bad in (dict(rows=0), dict(rows=1 << 31), dict(heads=0), dict(heads=5)):
        refused(lambda: qkrope(pages(), **bad), -1, "out of range")
    for bad in (dict(qs=255), dict(ks=127), dict(vs=100)):
        refused(lambda: qkrope(pages(), **bad), -1, "stride below")
    refused(lambda: qkrope(pages(), qs=1 << 37), -1, "2^36")
    refused(lambda: qkrope(pages(), rows=(1 << 23) + 1), -1, "out of range")
    refused(lambda: qkrope(pages(), heads=1 << 60), -1, "out of range")
    refused(lambda: qkrope(pages(), q=A + 2), -1, "4 bytes")
    for bad in (-1.0, float("nan"), float("inf")):
        refused(lambda: qkrope(pages(), eps=bad), -1, "eps")
    for bad in (dict(freq=0), dict(freq=A, dims=7), dict(freq=A, dims=66), dict(freq=A, dims=-2)):
        refused(lambda: qkrope(pages(), H.Rope(**bad)), -1, "rope")
    refused(lambda: qkrope(pages(), H.Rope(freq=A, scale=float("nan"))), -1, "scale")
    refused(lambda: qkrope(pages(), H.Rope(freq=A, dims=10)), -1, "no context")


def test_slots_refused():
    def call(**kw):
        a = dict(past=A, count=0, seqs=3, table=A, max_pages=4, page_size=16, ring=A, pages=9,
                 ends=A, ends_out=A, offsets=A, lengths=A, positions=A, slots=A, rows=7, failed=0)
        a.update(kw)
        return H.lib().ihip_enqueue_paged_slots(None, *a.values())

    for name in ("past", "table", "ring", "ends", "ends_out", "offsets", "lengths", "positions",
                 "slots"):
        refused(lambda: call(**{name: 0}), -1, "missing array")
    for bad in (dict(seqs=0), dict(rows=0), dict(rows=1 << 31), dict(page_size=0), dict(pages=0),
                dict(pages=1 << 28), dict(max_pages=0), dict(max_pages=1 << 28),
                dict(page_size=1 << 32)):
        refused(lambda: call(**bad), -1, "out of range")
    refused(lambda: call(seqs=H.PAGED_SEQS + 1), -6, "IHIP_PAGED_SEQS")
    refused(lambda: call(ends=A + 4), -1, "8 bytes")
    refused(lambda: call(), -1, "no context")


def test_logprobs_refused():
    def call(**kw):
        a = dict(logits=A, rows=3, vocab=1000, stride=0, ids=A, logprobs=A, entropy=A, k=5,
                 top_ids=A, top_logprobs=A)
        a.update(kw)
        return H.lib().ihip_enqueue_logprobs(None, *a.values())

    for bad in (dict(logits=0), dict(ids=0), dict(top_ids=0), dict(top_logprobs=0),
                dict(logprobs=0, entropy=0, k=0)):
        refused(lambda: call(**bad), -1, "missing array")
    for bad in (dict(rows=0), dict(rows=1 << 31), dict(vocab=0), dict(vocab=(1 << 22) + 1)):
        refused(lambda: call(**bad), -1, "out of range")
    for bad in (dict(k=-1), dict(k=H.LOGPROBS_TOP + 1)):
        refused(lambda: call(**bad), -6, "IHIP_LOGPROBS_TOP")
    refused(lambda: call(stride=999), -1, "stride below")
    refused(lambda: call(stride=1 << 37), -1, "2^36")
    refused(lambda: call(entropy=A + 1), -1, "4 bytes")
    refused(lambda: call(ids=0, logprobs=0), -1, "no context")


# ------------------------------------------------------------- the arithmetic
def value(page, at, pages, page_stride, slot_stride):
    f = O.lib().orc_paged_value
    f.restype = C.c_int64
    f.argtypes = [C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.c_int64]
    return f(page, at, pages, page_stride, slot_stride)


def slot_value(slot, page_size, pages, page_stride, slot_stride):
    f = O.lib().orc_paged_slot_value
    f.restype = C.c_int64
    f.argtypes = [C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.c_int64]
    return f(slot, page_size, pages, page_stride, slot_stride)


def key_range(length, window, max_pages, page_size):
    f = O.lib().orc_paged_range
    f.restype = None
    f.argtypes = [C.c_int32, C.c_int64, C.c_int64, C.c_int32, C.c_void_p, C.c_void_p]
    lo, hi = C.c_int64(), C.c_int64()
    f(length, window, max_pages, page_size, C.byref(lo), C.byref(hi))
    return lo.value, hi.value


@pytest.mark.parametrize("page", [-1, -2 ** 31, 8, 9, 2 ** 31 - 1])
def test_pages_outside_the_pool(page):
    assert value(page, 3, 8, 4096, 256) == -1


def test_values_beyond_32_bits():
    assert value(70000, 5, 70001, 1 << 20, 1024) == 70000 * 2 ** 20 + 5 * 1024
    assert value(0, 0, 1, 1, 1) == 0
    assert slot_value(2 ** 31 - 1, 1, 2 ** 31 - 1, 8, 8) == -1  # the page behind the last
    assert slot_value(2 ** 31 - 2, 1, 2 ** 31 - 1, 8, 8) == (2 ** 31 - 2) * 8


@pytest.mark.parametrize("page_size", [1, 7, 16, 100])
def test_slots_are_pages_and_tokens(page_size):
    pages, ps, ss = 9, 3 * 64 * page_size, 192
    for slot in range(pages * page_size):
        assert slot_value(slot, page_size, pages, ps, ss) == \
            slot // page_size * ps + slot % page_size * ss
    for slot in (-1, -page_size, pages * page_size, pages * page_size + 1, 2 ** 31 - 1):
        assert slot_value(slot, page_size, pages, ps, ss) == -1


@pytest.mark.parametrize("length", [-2 ** 31, -1, 0, 1, 15, 16, 17, 63, 64, 65, 2 ** 31 - 1])
@pytest.mark.parametrize("window", [0, 1, 16, 100, 2 ** 40])
def test_ranges_stay_in_the_table(length, window):
    lo, hi = key_range(length, window, 4, 16)
    n = min(max(length, 0), 64)
    assert (lo, hi) == (max(0, n - window) if window else 0, n)


# --------------------------------------------------------------- the oracle
def test_plan_oracle():
    table = np.full((4, 3), -1, np.int32)
    table[0, :1], table[1, :2], table[2, :1] = 5, (7, 2), 3
    got = R.slots(np.array([4, 5, 3, -1]), np.array([1, -1, 2, 4]), table, 4,
                  np.array([9, 8, 6, 4, 1, 0, 0, 0, 0, 0], np.int32), (0, 6), 8)
    assert got["positions"].tolist() == [4, 3, 4, -1, -1, -1, -1, -1]
    assert got["slots"].tolist() == [9 * 4, 3 * 4 + 3, 8 * 4, -1, -1, -1, -1, -1]
    assert got["lengths"].tolist() == [5, -1, 5, -1] and got["ends"].tolist() == [2, 8]
    assert got["ring"][6:8].tolist() == [7, 2] and got["offsets"].tolist() == [0, 1, 1, 3, 3]


def test_attention_oracle_matches_softmax():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 3, 4, 1, 8))
    q = rng.standard_normal((1, 2, 8))
    y, tol = R.attention(q, k, v, np.array([[2, 0]]), [7], 4)
    kk = np.concatenate([k[2], k[0, :3]])[:, 0]
    vv = np.concatenate([v[2], v[0, :3]])[:, 0]
    p = np.exp(kk @ q[0].T / 8 ** 0.5)
    assert np.allclose(y[0], (p / p.sum(0)).T @ vv, rtol=1e-14, atol=0)
    assert (tol > 0).all() and tol.max() < 1e-4


@pytest.mark.parametrize("name", ["qwen3-0.6b-q8_0", "gpt-oss-20b-mxfp4"])
def test_frequencies_are_the_tables(name):
    spec = models.Spec(models.tiny(name, layers=1, vocab=64), seed=3)
    half = spec.cfg["head_dim"] // 2
    f, scale = np.empty(half, np.float32), C.c_double()
    H.check(H.lib().ihip_model_frequencies(C.addressof(spec.struct), f.ctypes.data, C.byref(scale)))
    cs = np.empty(4 * half, np.float32)
    H.check(H.lib().ihip_model_rotary(C.addressof(spec.struct), 1, 2, cs.ctypes.data))
    # cos, then sin, of the frequencies: rounded, then times the scale, rounded
    want = np.concatenate([np.cos(f.astype(np.float64)), np.sin(f.astype(np.float64))])
    got = np.concatenate([cs[:half], cs[2 * half:3 * half]])
    assert np.all(np.abs(got - want * scale.value) <= 2 * 2.0 ** -24 * np.abs(want) * 2)
    H.check(H.lib().ihip_model_frequencies(C.addressof(spec.struct), f.ctypes.data, None))
    refused(lambda: H.lib().ihip_model_frequencies(None, f.ctypes.data, None), -1, "frequencies")

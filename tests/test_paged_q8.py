"""8-bit pages on the host (no device): refused pools and calls, and the wait states of
the matrix products in the code object that the build made of csrc/kernels/paged_q8.hip."""
import ctypes as C
import os

import pytest

import infer_hip as H
from code_objects import OBJDUMP, build_of, products_wait
from test_paged import A, attention, pages, qkrope, refused


def q8(**kw):
    a = dict(dtype=H.Q8_HEAD, k_scale=A, v_scale=A)
    a.update(kw)
    return pages(**a)


BAD = [
    (dict(k_scale=0), -1, "without scales"), (dict(v_scale=0), -1, "without scales"), (dict(v_scale=A + 2), -1, "without scales"),
    (dict(head_dim=72), -3, "multiple of 16"), (dict(head_dim=8), -3, "multiple of 16"),
    (dict(slot_stride=144), -1, "no multiple of head_dim"), (dict(page_stride=16 * 128 + 16), -1, "no multiple of head_dim"),
    (dict(head_stride=80), -1, "no multiple of head_dim"), (dict(slot_stride=130), -1, "16 bytes"), (dict(k=A + 8), -1, "aligned"),
]


def read(pool, **kw):
    a = dict(table=A, mp=4, first=0, offsets=A, seqs=3, rows=50, out=H.F32, k=A + (1 << 24), v=A + (1 << 25))
    a.update(kw)
    return H.lib().ihip_enqueue_paged_read(None, C.byref(pool) if pool is not None else None, *a.values())


@pytest.mark.parametrize("bad,rc,text", BAD)
def test_pools_refused(bad, rc, text):
    for call in (attention, qkrope, read):
        refused(lambda: call(q8(**bad)), rc, text)


def test_in_order_but_the_context():
    for call in (attention, qkrope, read):
        refused(lambda: call(q8()), -1, "no context")
        refused(lambda: call(q8(slot_stride=64, head_stride=1024)), -1, "no context")


def test_read_refused():
    refused(lambda: read(None), -1, "no cache")
    for name in ("table", "offsets", "k", "v"):
        refused(lambda: read(q8(), **{name: 0}), -1, "missing array")
    for out in (H.BF16, H.Q8_0, 0, H.Q8_HEAD):
        refused(lambda: read(q8(), out=out), -3, "F32 or F16")
    for bad in (dict(seqs=0), dict(rows=0), dict(rows=1 << 31), dict(mp=0), dict(mp=1 << 28)):
        refused(lambda: read(q8(), **bad), -1, "out of range")
    refused(lambda: read(q8(), seqs=H.PAGED_SEQS + 1), -6, "IHIP_PAGED_SEQS")
    for bad in (dict(table=A + 2), dict(first=A + 1), dict(offsets=A + 3)):
        refused(lambda: read(q8(), **bad), -1, "4 bytes")
    refused(lambda: read(q8(), k=A + (1 << 24) + 8), -1, "16 bytes")
    # the rows (50 of 2 heads of 64) against each other, the pool (8 pages of 16) and its scales
    B, n, held = A + (1 << 24), 50 * 2 * 64 * 4, 8 * 16 * 2 * 64
    refused(lambda: read(q8(), v=B + n - 16), -1, "overlap")
    refused(lambda: read(q8(), v=B - n + 16), -1, "overlap")
    refused(lambda: read(q8(), v=B + n), -1, "no context")
    refused(lambda: read(q8(), k=A - n + 16), -1, "overlap")
    refused(lambda: read(q8(), k=A - n), -1, "no context")
    refused(lambda: read(q8(k=4 * A, v=8 * A, k_scale=B, v_scale=4 * B), k=B - n + 16, v=2 * B), -1, "overlap")
    refused(lambda: read(q8(k=4 * A, v=8 * A, k_scale=4 * B, v_scale=B), k=3 * B, v=B + held // 64 * 4 - 16), -1, "overlap")
    refused(lambda: read(q8(k=4 * A, v=8 * A, k_scale=4 * B, v_scale=B), k=3 * B, v=B + held // 64 * 4), -1, "no context")
    # other pools' scale fields are not looked at
    refused(lambda: read(pages(k_scale=B, v_scale=B)), -1, "no context")


@pytest.mark.skipif(not os.path.exists(build_of("paged_q8")) or not os.path.exists(OBJDUMP),
                    reason="no code object or disassembler")
def test_products_wait(tmp_path):
    assert products_wait("paged_q8", tmp_path) > 8 * 8

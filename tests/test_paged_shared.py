"""Attention of groups that share their first tokens, on the host (no device): refused
calls, what a group has in common, and the wait states of the kernels' products."""
import ctypes as C
import os

import pytest

import infer_hip as H
import oracle_lib as O
from code_objects import OBJDUMP, build_of, products_wait
from test_paged import A, pages, refused


def call(pool=None, **kw):
    a = dict(ctx=None, q=A, qs=0, pool=pool or C.byref(pages()), table=A, mp=4, lengths=A, offsets=0, rows=3, members=A,
             shared=A, groups=2, y=8 * A, seqs=3, heads=4, window=0, sinks=0, scale=0.0)
    a.update(kw)
    return H.lib().ihip_enqueue_paged_attention_shared(*a.values())


def test_refused():
    refused(lambda: call(C.byref(pages(dtype=H.Q8_0))), -3, "F32, F16 or BF16")
    refused(lambda: call(C.byref(pages(dtype=H.Q8_HEAD))), -1, "without scales")
    for name in ("q", "table", "lengths", "y", "members", "shared"):
        refused(lambda: call(**{name: 0}), -1, "missing array")
        refused(lambda: call(**{name: 16 * A + 2}), -1, "aligned")
    for bad in (dict(seqs=0), dict(heads=3), dict(heads=65536), dict(window=-1), dict(mp=0), dict(rows=0), dict(rows=1 << 31)):
        refused(lambda: call(**bad), -1, "out of range")
    for groups in (0, -1, 4):
        refused(lambda: call(groups=groups), -1, "groups out of range")
    refused(lambda: call(seqs=H.PAGED_SEQS + 1), -6, "IHIP_PAGED_SEQS")
    refused(lambda: call(seqs=4096, heads=258, rows=4096, mp=1), -6, "2^20 heads")
    refused(lambda: call(seqs=4096, heads=256, rows=4096, mp=1, y=1 << 40), -1, "no context")
    refused(lambda: call(qs=255), -1, "stride below")
    for bad in (-1.0, float("nan"), 3e38):
        refused(lambda: call(scale=bad), -1, "scale")
    # y is refused wherever it meets q, its own rows among them
    refused(lambda: call(y=A), -1, "overlaps q")
    refused(lambda: call(y=A + 3 * 4 * 64 * 4 - 4), -1, "overlaps q")
    refused(lambda: call(y=A + 3 * 4 * 64 * 4), -1, "no context")
    refused(lambda: call(), -1, "no context")
    refused(lambda: call(window=100), -1, "no context")


def test_common_tokens():
    f = O.lib().orc_paged_common
    f.restype, f.argtypes = C.c_int64, [C.c_int32] * 4 + [C.c_int64, C.c_int32]
    most = 2 ** 31 - 1
    assert f(0, 2, 5, 3, 4, 16) == 5 and f(1, 3, 64, 3, 4, 16) == 64
    assert f(1, 3, 65, 3, 4, 16) == 64 and f(0, 3, most, 3, 4, 16) == 64  # the tables' width
    assert f(0, 3, most, 3, most, 1) == most
    # one sequence, none, a group that ends before it begins or outside the batch, no tokens
    for first, end, shared in ((0, 1, 5), (2, 2, 5), (2, 1, 5), (-1, 2, 5), (-2 ** 31, most, 5), (most, -2 ** 31, 5),
                               (1, 4, 5), (0, most, 5), (0, 2, 0), (0, 2, -1), (0, 2, -2 ** 31)):
        assert f(first, end, shared, 3, 4, 16) == 0


@pytest.mark.parametrize("name", ["f32", "f16", "bf16", "q8"])
def test_products_wait(name, tmp_path):
    name = "paged_shared_" + name
    if not os.path.exists(build_of(name)) or not os.path.exists(OBJDUMP):
        pytest.skip("no code object or disassembler")
    assert products_wait(name, tmp_path) > 16 * 8

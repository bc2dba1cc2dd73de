"""The paged operators on the host (no device), at the edges of what a call may
hold: rows beyond the step's, refusals."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import oracle_lib as O
from infer_hip import models
from test_paged import A, attention, pages, qkrope, refused


def row(first, end, rows):
    f = O.lib().orc_paged_row
    f.restype = C.c_int32
    f.argtypes = [C.c_int32, C.c_int32, C.c_int32]
    return f(first, end, rows)


@pytest.mark.parametrize("rows", [1, 2, 7, 2 ** 31 - 1])
def test_rows_stay_in_the_step(rows):
    """A sequence's row is the last of its own, and never one that the arrays do not have."""
    low, high = -2 ** 31, 2 ** 31 - 1
    for first in (low, -1, 0, 1, 5, 6, high - 1, high):
        for end in (low, -1, 0, 1, 2, 6, 7, 8, high):
            r = row(first, end, rows)
            assert r == (end - 1 if end > first and 1 <= end <= rows else -1), (first, end)
            assert -1 <= r < rows


def test_rows_without_offsets():
    """Row s of sequence s, where there is one."""
    assert [row(s, s + 1, 3) for s in range(6)] == [0, 1, 2, -1, -1, -1]


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("scale", [-0.125, -1e-300, 1e39, 3e38])
def test_attention_scales_refused(scale):
    """A scale below 0 (which no formula here has: 0 alone stands for the default), and one that
    leaves single when the exponential's base is 2."""
    refused(lambda: attention(pages(), scale=scale), -1, "scale")


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-30, 2.3e38])
def test_attention_scales_taken(scale):
    refused(lambda: attention(pages(), scale=scale), -1, "no context")


@pytest.mark.parametrize("skew", [1, 2, 3])
def test_unaligned_numbers_refused(skew):
    """Lengths, tables, positions and slots are int32, aligned to 4 bytes, as the attention's are."""
    names = ("past", "count", "seqs", "table", "max_pages", "page_size", "ring", "pages", "ends", "ends_out", "offsets",
             "lengths", "positions", "slots", "rows", "failed")
    good = dict(zip(names, (A, A, 3, A, 4, 16, A, 9, A, A, A, A, A, A, 7, A)))

    def slots(**kw):
        return H.lib().ihip_enqueue_paged_slots(None, *dict(good, **kw).values())

    refused(slots, -1, "no context")
    for name in ("past", "count", "table", "ring", "offsets", "lengths", "positions", "slots", "failed"):
        refused(lambda: slots(**{name: A + skew}), -1, "4 bytes")
    for name in ("positions", "slots"):
        refused(lambda: qkrope(pages(), **{name: A + skew}), -1, "4 bytes")


@pytest.mark.parametrize("dims,head_dim", [(66, 64), (2 ** 31 - 2, 64), (0, 514), (514, 514), (0, 2 ** 31 - 2), (0, 0),
                                           (0, -64), (0, 63), (63, 64)])
def test_frequencies_refused(dims, head_dim):
    """The shares of a head that a model is refused for, before anything of their size is allocated."""
    spec = models.Spec(models.tiny("qwen3-0.6b-q8_0", layers=1, vocab=64), seed=3)
    spec.struct.rope_dims, spec.struct.head_dim = dims, head_dim
    f = np.zeros(256, np.float32)
    refused(lambda: H.lib().ihip_model_frequencies(C.addressof(spec.struct), f.ctypes.data, None), -1, "frequencies")
    assert (f == 0).all()


# (addresses of rows of 4 heads of 64 and 2 KV heads each of k and v: 256, 128 and 128 floats)
W = 4 * 512


@pytest.mark.parametrize("where,strides,ok", [
    (A, 0, True), (A, 512, False), (A + 1024, 0, False), (A - 1024, 0, False), (A + 4, 0, False),
    (A + 5 * 1024, 0, True), (A - 5 * 1024, 0, True), (A + W - 4, 512, False), (A + 5 * W, 512, True),
    (A + 4 * W + 3 * 512, 512, False), (A + 4 * W + 4 * 512, 512, True), (A + 2048, 2048, True), (A + 1024, 2048, False),
    (A + 8192 - 5 * 1024, 2048, True), (A + 8192 - 5 * 1024 + 4, 2048, False), (A + 4 * 8192 + 2048, 2048, True)])
def test_qkrope_outputs_over_inputs(where, strides, ok):
    """q_out is q's own rows, contiguous, or apart from q, k and v: rows of a call are turned at once."""
    kw = dict(qs=strides, ks=strides, vs=strides, k=A + 1024, v=A + 1536) if strides else dict(k=A << 1, v=A << 2)
    refused(lambda: qkrope(pages(), out=where, **kw), -1, "no context" if ok else "q_out")


def test_qkrope_output_over_keys():
    for name in ("k", "v"):
        refused(lambda: qkrope(pages(), q=A << 3, k=A << 4, v=A << 5, out=(A << (4 if name == "k" else 5)) + 512), -1, "q_out")
    refused(lambda: qkrope(pages(), q=A << 3, k=A << 4, v=A << 5, out=A << 6), -1, "no context")


@pytest.mark.parametrize("where,stride,ok", [
    (A, 0, True), (A, 256, True), (A, 512, False), (A + 1024, 0, False), (A - 1024, 256, False), (A + 3 * 1024, 0, True),
    (A - 3 * 1024, 0, True), (A + 1024, 512, False), (A + 1024, 1024, True), (A + 2 * 4096 + 1024, 1024, True)])
def test_attention_output_over_queries(where, stride, ok):
    """y is q's own rows, contiguous, or apart from them."""
    refused(lambda: attention(pages(), y=where, q_stride=stride), -1, "no context" if ok else "y overlaps")

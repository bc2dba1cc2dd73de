"""A batch served over 8-bit pages with prompts in common: each step the last tokens' rows of a
table as q, k and v, the plan, the store, attention with the prompts read once for their
groups, logits and a draw for every row, whose tokens are the next step's. Eager and
captured; every step against its definition in 64 bits on the histories read back."""
import ctypes as C

import numpy as np
import pytest

import infer_hip as H
import paged_ref as R
import sample_ref as S
from test_gpu_paged import assert_close, ctx, dev  # noqa: F401 (fixtures)
from test_gpu_paged_q8 import q8_pool
from test_gpu_sample_rows import settings_array

pytestmark = pytest.mark.gpu
U = R.U
HD, HEADS, KVH, PS, WIDTH, VOCAB = 64, 8, 2, 8, 24, 700
GROUPS = [(3, 40), (1, 16), (3, 8)]  # sequences, tokens that their prompts have in common (whole pages)
N = 7
STEPS = 6
SETTINGS = [(0.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05),
            (1.0, 5, 1.0, 0.1), (0.0, 3, 0.5, 0.0)]
ROW = (HEADS + 2 * KVH) * HD


class Batch:
    def __init__(self, ctx, dev):
        rng = np.random.default_rng(77)
        self.ctx, self.L = ctx, H.lib()
        self.embed = rng.standard_normal((VOCAB, ROW)).astype(np.float32)
        self.head = (rng.standard_normal((VOCAB, HEADS * HD)) * 0.1).astype(np.float32)
        self.uniform = rng.random((STEPS, N))
        past = np.repeat([g[1] for g in GROUPS], [g[0] for g in GROUPS]).astype(np.int32)
        pages = 60
        ring, table, at, slots = rng.permutation(pages).astype(np.int32), np.full((N, WIDTH), -1, np.int32), 0, []
        first = np.cumsum([0] + [g[0] for g in GROUPS])
        for (n, common), m in zip(GROUPS, first):  # the prompts' pages, from the ring's start
            for p in range(common // PS):
                table[m:m + n, p] = ring[at]
                slots += [ring[at] * PS + t for t in range(PS)]
                at += 1
        self.past, self.lengths = past, past.copy()
        freq = (1.0 / 10000.0 ** (np.arange(0, HD, 2) / HD)).astype(np.float32)
        self.rope = H.Rope(freq=dev(freq))
        self.bufs = [dev.out(pages * PS * KVH * HD) for _ in range(2)] + [dev.out(pages * PS * KVH * 4, 0xFF) for _ in range(2)]
        self.pool = q8_pool([b.ptr for b in self.bufs], pages, PS, KVH, HD)
        self.b = {}
        for name, a in dict(past=past, table=table, ring=ring, ends=np.array([at, pages], np.int64),
                            count=np.ones(N, np.int32), ids=rng.integers(0, VOCAB, N).astype(np.int32),
                            uniform=self.uniform[0]).items():
            self.b[name] = dev.out(a.nbytes)
            self.b[name].upload(a)
        self.pages = pages
        self.de, self.dw = dev(self.embed), dev(self.head)
        self.members, self.shared = dev(first.astype(np.int32)), dev(np.array([g[1] for g in GROUPS], np.int32))
        self.settings = dev(settings_array(SETTINGS))
        for name, n in dict(x=N * ROW * 4, y=N * HEADS * HD * 4, logits=N * VOCAB * 4, probs=4 * N, offsets=4 * N + 4,
                            positions=4 * N, slots=4 * N, failed=4).items():
            self.b[name] = dev.out(n)
        self.bound = N * WIDTH * PS
        self.every = dev(np.arange(0, self.bound + 1, WIDTH * PS, dtype=np.int32))
        self.back = [dev.out(self.bound * KVH * HD * 4) for _ in range(2)]
        # the prompts' own rows
        prompt = rng.standard_normal((len(slots), ROW)).astype(np.float32)
        where = np.concatenate([np.arange(g[1]) for g in GROUPS]).astype(np.int32)
        self.store(dev(prompt), len(slots), dev(where), dev(np.array(slots, np.int32)))

    def store(self, x, rows, positions, slots):
        H.check(self.L.ihip_enqueue_paged_qkrope(
            self.ctx.h, x, ROW, x + 4 * HEADS * HD, ROW, x + 4 * (HEADS + KVH) * HD, ROW, rows, HEADS, 0, 0, 0.0,
            C.byref(self.rope), positions, slots, C.byref(self.pool), 0))

    def enqueue(self):
        b, L, h = {n: v.ptr for n, v in self.b.items()}, self.L, self.ctx.h
        H.check(L.ihip_enqueue_embed(h, self.de, H.F32, VOCAB, ROW, b["ids"], N, b["x"]))
        H.check(L.ihip_enqueue_paged_slots(
            h, b["past"], b["count"], N, b["table"], WIDTH, PS, b["ring"], self.pages, b["ends"], b["ends"], b["offsets"],
            b["past"], b["positions"], b["slots"], N, b["failed"]))
        self.store(b["x"], N, b["positions"], b["slots"])
        H.check(L.ihip_enqueue_paged_attention_shared(
            h, b["x"], ROW, C.byref(self.pool), b["table"], WIDTH, b["past"], b["offsets"], N, self.members, self.shared,
            len(GROUPS), b["y"], N, HEADS, 0, 0, 0.0))
        H.check(L.ihip_enqueue_linear_at_static(h, b["y"], N, HEADS * HD, H.F32, self.dw, VOCAB, b["logits"], 0, H.MODE_F32))
        H.check(L.ihip_enqueue_sample_rows(h, b["logits"], N, VOCAB, 0, self.settings, b["uniform"], b["ids"], b["probs"]))

    def check(self, step, before):
        """One step's outputs: (tokens, probabilities, logits, attention)."""
        b = self.b
        self.lengths = self.lengths + 1
        assert np.array_equal(b["past"].download(np.int32, N), self.lengths) and b["failed"].download(np.int32, 1)[0] == 0
        x = b["x"].download(np.float32, N * ROW).reshape(N, ROW)
        v0 = (HEADS + KVH) * HD
        assert np.array_equal(x[:, v0:], self.embed[before][:, v0:])  # (q is turned in place)
        q = x[:, :HEADS * HD].reshape(N, HEADS, HD).astype(np.float64)
        H.check(self.L.ihip_enqueue_paged_read(self.ctx.h, C.byref(self.pool), b["table"].ptr, WIDTH, 0, self.every, N,
                                               self.bound, H.F32, self.back[0].ptr, self.back[1].ptr))
        k, v = (a.download(np.float32, self.bound * KVH * HD).reshape(N * WIDTH, PS, KVH, HD).astype(np.float64)
                for a in self.back)
        # the row that the step has stored: its values within half a step of the codes
        for s in range(N):
            at = self.lengths[s] - 1
            got, want = v[s * WIDTH + at // PS, at % PS], x[s, v0:].reshape(KVH, HD)
            assert (np.abs(got - want).max(1) <= np.abs(want).max(1) / 127 * (0.5 + 1e-5)).all()
        mine = np.arange(N * WIDTH).reshape(N, WIDTH).astype(np.int32)
        want, tol = R.attention(q, k, v, mine, self.lengths, PS)
        # values read back are codes times scales rounded to single, which the attention's are not: U of
        # each score's products and of each value; small weights are off by 2^-39 of the largest
        top_k, top = (max(np.abs(a.reshape(N, WIDTH * PS, KVH, HD)[s, :self.lengths[s]]).max() for s in range(N)) for a in (k, v))
        tol = tol + 4 * U * (top + top_k * np.abs(q).max() * HD * top) + 2.0 ** -39 * WIDTH * PS * top
        y = b["y"].download(np.float32, want.size).reshape(want.shape)
        assert_close(y, want, tol)
        # logits: HEADS HD products added up in single in any order
        logits = b["logits"].download(np.float32, N * VOCAB).reshape(N, VOCAB)
        w, yy = self.head.astype(np.float64), y.reshape(N, -1).astype(np.float64)
        assert_close(logits, yy @ w.T, (HEADS * HD + 2) * U * (np.abs(yy) @ np.abs(w).T))
        ids, probs = b["ids"].download(np.int32, N), b["probs"].download(np.float32, N)
        for s in range(N):
            want, prob, margin = S.draw(logits[s], *SETTINGS[s], self.uniform[step, s])
            if margin >= 1e-10:  # (weights are off by less)
                assert ids[s] == want and abs(probs[s] - prob) <= prob * (2.0 ** -24 + 1e-9), (step, s)
        return ids, probs, logits, y


def run(ctx, dev, graph):
    batch, out = Batch(ctx, dev), []
    if graph:
        H.check(batch.L.ihip_capture_begin(ctx.h))
        batch.enqueue()
        H.check(batch.L.ihip_capture_end(ctx.h, graph))
    for step in range(STEPS):
        before = batch.b["ids"].download(np.int32, N)
        batch.b["uniform"].upload(batch.uniform[step])
        if graph:
            H.check(batch.L.ihip_graph_launch(ctx.h, graph))
        else:
            batch.enqueue()
        out.append(batch.check(step, before))
    return out


def test_steps(ctx, dev):
    tokens = np.array([o[0] for o in run(ctx, dev, 0)])
    assert len(np.unique(tokens)) > STEPS  # (the draws differ from row to row)


def test_replayed_steps_are_the_eager_ones(ctx, dev):
    for a, b in zip(run(ctx, dev, 0), run(ctx, dev, 12)):
        for x, y in zip(a, b):
            assert np.array_equal(x, y)

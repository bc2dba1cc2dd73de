"""The measured work of a batched decode step: several sequences over one paged
key-value cache, and the scores of their tokens, through the C-ABI entry points
of infer_hip.

Four kinds of case:

- slots: the step's plan (block tables, positions and slots of the new rows) from
  the sequences' lengths, pages taken from and put back into the free ring;
- rope: head norms and rotary positions of the new rows' q and k, k and v stored
  into the pages; either pair layout, a part of the head, scaled frequencies;
- attention: one new token of each sequence over its pages;
- logprobs: log probabilities of given tokens, entropies and top alternatives.

The plain forms are elementary torch operations in 32 bits (64 for the angles of
far positions).
"""
import json
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step of 64 chats: one token each, a few of them ended
        dict(name="slots-decode", kind="slots", seqs=64, most=4096, new=1, page=16, rows=64),
        # prompts arriving beside running sequences, ragged, odd page size
        dict(name="slots-prompts", kind="slots", seqs=500, most=8192, new=700, page=24, rows=180000),
        # a decode step's rows, head norms (32 + 4 heads of 128)
        dict(name="rope-decode", kind="rope", rows=32, heads=32, kv_heads=4, head_dim=128, dims=128,
             interleaved=False, norm=True, scaled=False, most=8192, page=16, cache="f16"),
        # a batch of prompts, scaled frequencies and far positions (64 + 8 heads of 64)
        dict(name="rope-prompts", kind="rope", rows=8000, heads=64, kv_heads=8, head_dim=64, dims=64,
             interleaved=False, norm=False, scaled=True, most=131072, page=32, cache="bf16"),
        # a quarter of the head rotating, interleaved pairs, single cache, ragged rows
        dict(name="rope-partial", kind="rope", rows=1037, heads=8, kv_heads=2, head_dim=256, dims=64,
             interleaved=True, norm=True, scaled=False, most=32768, page=17, cache="f32"),
        # one chat after a 1151-token context: latency
        dict(name="attention-one", kind="attention", seqs=1, least=1152, most=1152, heads=32,
             kv_heads=4, head_dim=128, window=0, sinks=False, page=16, cache="f16"),
        # a serving batch of ragged lengths
        dict(name="attention-batch", kind="attention", seqs=64, least=1, most=4100, heads=16,
             kv_heads=8, head_dim=128, window=0, sinks=False, page=16, cache="bf16"),
        # a sliding-window layer with sinks
        dict(name="attention-window", kind="attention", seqs=48, least=60, most=9000, heads=64,
             kv_heads=8, head_dim=64, window=128, sinks=True, page=32, cache="f16"),
        # few long documents, heads of 256: the split over the length
        dict(name="attention-long", kind="attention", seqs=3, least=90000, most=131072, heads=8,
             kv_heads=2, head_dim=256, window=0, sinks=False, page=64, cache="f16"),
        # the chosen token of one chat with 20 alternatives: latency
        dict(name="logprobs-token", kind="logprobs", rows=1, vocab=151936, top=20),
        # a decode step's rows with 5 alternatives
        dict(name="logprobs-batch", kind="logprobs", rows=61, vocab=201088, top=5),
        # the scores of a whole prompt chunk
        dict(name="logprobs-prompt", kind="logprobs", rows=1024, vocab=151936, top=1),
    ]


HEADS = ((32, 4, 128), (16, 8, 128), (64, 8, 64), (8, 2, 256), (16, 8, 256), (14, 2, 64), (16, 2, 512),
         (12, 12, 96), (32, 2, 80), (48, 2, 128))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("slots", "rope", "attention", "logprobs"), (2, 3, 6, 3))[0]
    page = rng.choice((1, 7, 16, 24, 32, 64, 100, 128, 256))
    if kind == "slots":
        seqs, new = _log(rng, 1, 500), rng.choice((1, 1, _log(rng, 2, 700)))
        return dict(kind=kind, seqs=seqs, most=_log(rng, 64, 8192), new=new, page=page,
                    rows=seqs if new == 1 else min(seqs * new, 180000))
    heads, kv, hd = rng.choice(HEADS)
    cache = rng.choice(("f16", "f16", "bf16", "f32"))
    if kind == "rope":
        dims = rng.choice((hd, hd, hd // 2, max(2, hd // 4 // 2 * 2)))
        rows = _log(rng, 1, max(2, min(8000, 40000000 // ((heads + 2 * kv) * hd))))
        return dict(kind=kind, rows=rows, heads=heads, kv_heads=kv, head_dim=hd, dims=dims,
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
                    scaled=rng.random() < 0.5, most=_log(rng, 64, 131072), page=page, cache=cache)
    if kind == "attention":
        seqs = _log(rng, 1, 128)
        # at most the bytes of the largest listed case
        cap = int(600e6 / (seqs * 2 * kv * hd * 4))
        most = max(1, min(_log(rng, 16, 131072), cap))
        windowed = rng.random() < 0.3
        return dict(kind=kind, seqs=seqs, least=max(1, int(most * rng.choice((0.01, 0.3, 1.0)))),
                    most=most, heads=heads, kv_heads=kv, head_dim=hd,
                    window=rng.choice((128, 1000)) if windowed else 0, sinks=rng.random() < 0.3,
                    page=page, cache=cache)
    vocab = rng.choice((151936, 201088, 248320, 262144, _log(rng, 500, 200000)))
    rows = _log(rng, 1, max(2, min(1024, 150000000 // vocab)))
    return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice((1, 5, 20, 32)))


# ------------------------------------------------------------------- prepare
class State:
    pass


def _rand(c, seed):
    g = torch.Generator("cuda").manual_seed(seed * 7919 + len(c["kind"]))

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").int()

    return ints, normal, shuffled


def _tables(past, pages_of, width, order):
    """Block tables [seqs, width] that take the pages of `order` in turn, -1 behind them; how
    many they take."""
    first = torch.cumsum(pages_of, 0) - pages_of
    j = torch.arange(width, device="cuda")[None]
    at = (first[:, None] + j).clamp(max=len(order) - 1)
    return torch.where(j < pages_of[:, None], order[at], -1).int().contiguous()


def _slots_inputs(c, seed):
    ints, _, shuffled = _rand(c, seed)
    n, ps = c["seqs"], c["page"]
    past = ints(0, c["most"] - c["new"], n) if c["most"] > c["new"] else ints(0, 0, n)
    count = ints(1, c["new"], n) if c["new"] > 1 else torch.ones_like(past)
    # about one in 16 has ended, one in 16 is an empty place of the batch
    r = ints(0, 15, n)
    count = torch.where(r == 0, -1, count)
    past = torch.where((r == 1) & (n > 1), -1, past)
    width = -(-c["most"] // ps) + 1
    have = (past.clamp(min=0) + ps - 1) // ps
    taken = n * -(-c["most"] // ps)  # a pool that holds them all
    pages = taken + n * (-(-c["new"] // ps) + 1)
    order = shuffled(pages)
    used = int(have.sum())
    table = _tables(past, have, width, order)
    ring = torch.roll(order, -used).contiguous()  # the free pages from entry 0 on
    ends = torch.tensor([0, pages - used], dtype=torch.int64, device="cuda")
    return past.int(), count.int(), table, ring, ends


def _freqs(c):
    """The frequencies of the rotating pairs; scaled: the low ones slowed 32 times (YaRN's ramp
    between pairs that turn 32 times and once in 4096 positions) and the attention factor."""
    d = c["dims"]
    f = 1.0 / 150000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    if not c["scaled"]:
        return f.float(), 1.0
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return (f * keep + f / 32 * (1 - keep)).float(), 0.1 * math.log(32.0) + 1.0


def _rope_inputs(c, seed):
    ints, normal, shuffled = _rand(c, seed)
    n, hs, kv, hd, ps = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    # a fused product's rows: q, k and v of a row beside each other
    qkv = normal(n, (hs + 2 * kv) * hd)
    qn, kn = (1 + 0.1 * normal(hd), 1 + 0.1 * normal(hd)) if c["norm"] else (None, None)
    positions = ints(0, c["most"] - 1, n)
    pages = n // ps + 2
    slots = shuffled(pages * ps)[:n].contiguous()
    pool = [normal(pages, ps, kv, hd).to(DTYPES[c["cache"]]) for _ in range(2)]
    return qkv, qn, kn, positions, slots, pool[0], pool[1]


def _lengths(c, ints):
    return ints(c["least"], c["most"], c["seqs"])


def _attention_inputs(c, seed):
    ints, normal, shuffled = _rand(c, seed)
    kv, hd, ps, dt = c["kv_heads"], c["head_dim"], c["page"], DTYPES[c["cache"]]
    lengths = _lengths(c, ints)
    have = (lengths + ps - 1) // ps
    # half as many pages again as the sequences use: other sequences' keys
    used = int(have.sum())
    order = shuffled(used + used // 2 + 1)
    table = _tables(lengths, have, -(-c["most"] // ps), order)
    k, v = (normal(len(order), ps, kv, hd, dtype=dt) for _ in range(2))
    q = normal(c["seqs"], c["heads"], hd)
    return q, k, v, table, lengths, normal(c["heads"]) if c["sinks"] else None


def _logprobs_inputs(c, seed):
    ints, normal, _ = _rand(c, seed)
    x = normal(c["rows"], c["vocab"])
    x *= 2.5
    # a few likely tokens, as a trained head gives them
    at = ints(0, c["vocab"] - 1, c["rows"], 6).long()
    x.scatter_(1, at, normal(c["rows"], 6).abs() * 4 + 8)
    ids = torch.where(ints(0, 3, c["rows"]) > 0, at[:, 0].int(), ints(0, c["vocab"] - 1, c["rows"]))
    return x, ids.int().contiguous()


_handle = None


def _ctx():
    """The library and its device context, opened once, as a host does."""
    global _handle
    if _handle is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "mormot2-ai_amd"))
        import infer_hip as H
        _handle = (H, H.Context(0))
    return _handle


def _pages(H, k, v):
    return H.Pages(k=k.data_ptr(), v=v.data_ptr(), pages=k.shape[0], page_size=k.shape[1],
                   kv_heads=k.shape[2], head_dim=k.shape[3],
                   dtype={torch.float32: H.F32, torch.float16: H.F16, torch.bfloat16: H.BF16}[k.dtype])


def prepare(case, seed):
    c, s = case, State()
    s.case = c

    def i32(*n):
        return torch.zeros(n, dtype=torch.int32, device="cuda")

    if c["kind"] == "slots":
        s.past, s.count, s.table, s.ring, s.ends = _slots_inputs(c, seed)
        s.ends_out = torch.zeros_like(s.ends)
        s.offsets, s.lengths, s.failed = i32(c["seqs"] + 1), i32(c["seqs"]), i32(1)
        s.positions, s.slots = i32(c["rows"]), i32(c["rows"])
    elif c["kind"] == "rope":
        s.qkv, s.qn, s.kn, s.positions, s.slots, s.k, s.v = _rope_inputs(c, seed)
        s.freq, s.scale = _freqs(c)
        s.q_out = torch.zeros((c["rows"], c["heads"], c["head_dim"]), device="cuda")
    elif c["kind"] == "attention":
        s.q, s.k, s.v, s.table, s.lengths, s.sinks = _attention_inputs(c, seed)
        s.y = torch.zeros_like(s.q)
    else:
        s.x, s.ids = _logprobs_inputs(c, seed)
        s.lp, s.ent = (torch.zeros(c["rows"], device="cuda") for _ in range(2))
        s.top_ids = i32(c["rows"], c["top"])
        s.top_lp = torch.zeros((c["rows"], c["top"]), device="cuda")
    if own:
        H, s.ctx = _ctx()
        s.h = H
        if c["kind"] in ("rope", "attention"):
            s.pages = _pages(H, s.k, s.v)
        if c["kind"] == "rope":
            s.rope = H.Rope(freq=s.freq.data_ptr(), dims=c["dims"],
                            interleaved=int(c["interleaved"]), scale=s.scale)
    torch.cuda.synchronize()
    return s


# ----------------------------------------------------------------- one pass
def _slots_plain(s):
    c = s.case
    n, ps, width = c["seqs"], c["page"], s.table.shape[1]
    live = s.past >= 0
    ended = live & (s.count < 0)
    past = s.past.clamp(min=0).long()
    new = torch.where(live, s.count.clamp(min=0).long(), 0)
    offsets = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = torch.cumsum(new, 0)
    have = (past + ps - 1) // ps
    need = (past + new + ps - 1) // ps
    fits = (need <= width) & (offsets[1:] <= c["rows"])
    want = torch.where(fits & ~ended & live, need - have, 0)
    upto = torch.cumsum(want, 0)
    first, last = s.ends[0], s.ends[1]
    fits &= (upto <= last - first) | (want == 0)
    want = torch.where(fits, want, 0)
    first_of = upto - want
    pages = len(s.ring)
    # the new pages, in the sequences' order
    j = torch.arange(width, device="cuda")[None]
    fresh = (j >= have[:, None]) & (j < (have + want)[:, None])
    at = (first + first_of[:, None] + j - have[:, None]) % pages
    s.table.copy_(torch.where(fresh, s.ring[at], s.table))
    # the ended sequences' pages behind the free ones
    back = torch.where(ended, have.clamp(max=width), 0)
    back_at = torch.cumsum(back, 0) - back
    put = j < back[:, None]
    to = (last + back_at[:, None] + j) % pages
    s.ring[to[put]] = s.table[put]
    s.ends_out[0] = first + want.sum()
    s.ends_out[1] = last + back.sum()
    # the rows
    r = torch.arange(c["rows"], device="cuda")
    q = torch.searchsorted(offsets[1:], r, right=True).clamp(max=n - 1)
    there = r < offsets[n]
    pos = past[q] + r - offsets[q]
    page = s.table[q, (pos // ps).clamp(max=width - 1)].long()
    ok = there & fits[q] & (page >= 0)
    s.positions.copy_(torch.where(there, pos, -1))
    s.slots.copy_(torch.where(ok, page * ps + pos % ps, -1))
    s.offsets.copy_(offsets)
    s.lengths.copy_(torch.where(live & ~ended, past + torch.where(fits, new, 0), -1))
    s.failed[0] = (live & ~ended & ~fits).sum()
    return {"table": s.table, "ring": s.ring, "ends": s.ends_out, "offsets": s.offsets,
            "lengths": s.lengths, "positions": s.positions, "slots": s.slots, "failed": s.failed}


def _rope_plain(s):
    c = s.case
    n, hs, kv, hd, d = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["dims"]
    x = s.qkv.view(n, hs + 2 * kv, hd)
    q, k, v = x[:, :hs], x[:, hs:hs + kv], x[:, hs + kv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s.qn
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s.kn
    angle = s.positions.double()[:, None] * s.freq.double()
    cos, sin = ((t * s.scale).float()[:, None] for t in (angle.cos(), angle.sin()))

    def turn(t):
        if c["interleaved"]:
            a, b = t[..., 0:d:2], t[..., 1:d:2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = t[..., :d // 2], t[..., d // 2:d]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((r, t[..., d:]), -1)

    s.q_out.copy_(turn(q))
    at = s.slots.long()
    s.k.view(-1, kv, hd)[at] = turn(k).to(s.k.dtype)
    s.v.view(-1, kv, hd)[at] = v.to(s.v.dtype)
    return {"q": s.q_out, "k": s.k, "v": s.v}


def _attention_plain(s):
    c = s.case
    n, hs, kv, hd, ps = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    width = s.table.shape[1]
    # sequences in groups whose gathered keys stay small
    step = max(1, int(2e9 / (width * ps * kv * hd * 4)))
    for i in range(0, n, step):
        t, ln = s.table[i:i + step].long().clamp(min=0), s.lengths[i:i + step].long()
        m = t.shape[0]
        k = s.k[t].view(m, width * ps, kv, hd).permute(0, 2, 3, 1).float().contiguous()
        q = s.q[i:i + step].view(m, kv, hs // kv, hd) * hd ** -0.5
        x = q @ k
        del k
        j = torch.arange(width * ps, device="cuda")[None]
        seen = j < ln[:, None]
        if c["window"]:
            seen &= j >= ln[:, None] - c["window"]
        x = x.masked_fill(~seen[:, None, None], -math.inf)
        top = x.amax(-1, keepdim=True)
        if c["sinks"]:
            sink = s.sinks.view(1, kv, hs // kv, 1)
            top = torch.maximum(top, sink)
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True)
        if c["sinks"]:
            total = total + torch.exp(sink - top)
        v = s.v[t].view(m, width * ps, kv, hd).permute(0, 2, 1, 3).float().contiguous()
        s.y[i:i + step] = (p @ v / total).view(m, hs, hd)
    return s.y


def _logprobs_plain(s):
    c = s.case
    m = s.x.amax(1, keepdim=True)
    d = s.x - m
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    s.lp.copy_(d.gather(1, s.ids.long()[:, None])[:, 0] - log_total)
    s.ent.copy_(log_total - (d * e).sum(1) / total)
    for j in range(c["top"]):  # the first index of the largest value, again and again
        at = d.argmax(1, keepdim=True)
        s.top_ids[:, j] = at[:, 0].int()
        s.top_lp[:, j] = d.gather(1, at)[:, 0] - log_total
        d.scatter_(1, at, -math.inf)
    return {"logprobs": s.lp, "entropy": s.ent, "top_ids": s.top_ids, "top_logprobs": s.top_lp}


def run(s):
    c = s.case
    if not own:
        return {"slots": _slots_plain, "rope": _rope_plain, "attention": _attention_plain,
                "logprobs": _logprobs_plain}[c["kind"]](s)
    H, h = s.h, s.ctx.h
    L = H.lib()
    if c["kind"] == "slots":
        H.check(L.ihip_enqueue_paged_slots(
            h, s.past.data_ptr(), s.count.data_ptr(), c["seqs"], s.table.data_ptr(),
            s.table.shape[1], c["page"], s.ring.data_ptr(), len(s.ring), s.ends.data_ptr(),
            s.ends_out.data_ptr(), s.offsets.data_ptr(), s.lengths.data_ptr(),
            s.positions.data_ptr(), s.slots.data_ptr(), c["rows"], s.failed.data_ptr()), "slots")
        return {"table": s.table, "ring": s.ring, "ends": s.ends_out, "offsets": s.offsets,
                "lengths": s.lengths, "positions": s.positions, "slots": s.slots,
                "failed": s.failed}
    if c["kind"] == "rope":
        hs, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
        q, stride = s.qkv.data_ptr(), (hs + 2 * kv) * hd
        H.check(L.ihip_enqueue_paged_qkrope(
            h, q, stride, q + 4 * hs * hd, stride, q + 4 * (hs + kv) * hd, stride, c["rows"], hs,
            s.qn.data_ptr() if c["norm"] else 0, s.kn.data_ptr() if c["norm"] else 0, 1e-6,
            H.C.byref(s.rope), s.positions.data_ptr(), s.slots.data_ptr(), H.C.byref(s.pages),
            s.q_out.data_ptr()), "qkrope")
        return {"q": s.q_out, "k": s.k, "v": s.v}
    if c["kind"] == "attention":
        H.check(L.ihip_enqueue_paged_attention(
            h, s.q.data_ptr(), 0, H.C.byref(s.pages), s.table.data_ptr(), s.table.shape[1],
            s.lengths.data_ptr(), s.y.data_ptr(), c["seqs"], c["heads"], c["window"],
            s.sinks.data_ptr() if c["sinks"] else 0, 0.0), "attention")
        return s.y
    H.check(L.ihip_enqueue_logprobs(
        h, s.x.data_ptr(), c["rows"], c["vocab"], 0, s.ids.data_ptr(), s.lp.data_ptr(),
        s.ent.data_ptr(), c["top"], s.top_ids.data_ptr(), s.top_lp.data_ptr()), "logprobs")
    return {"logprobs": s.lp, "entropy": s.ent, "top_ids": s.top_ids, "top_logprobs": s.top_lp}


# --------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "slots":
        # the lengths, the plan's rows, and a table entry read for each page of the rows
        rows = min(c["rows"], int(c["seqs"] * (c["new"] + 1) / 2 * 14 / 16))
        return {"bytes": 16 * c["seqs"] + 8 * c["rows"] + 8 * (rows // c["page"] + c["seqs"]),
                "flops": 0}
    if c["kind"] == "rope":
        qw, kw = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        es = DTYPES[c["cache"]].itemsize
        return {"bytes": c["rows"] * (8 * qw + (8 + 2 * es) * kw + 8),
                "flops": c["rows"] * (qw + kw) * (6.0 if c["norm"] else 3.0)}
    if c["kind"] == "attention":
        # (the mean length: a case's own lengths follow the seed)
        keys = (c["least"] + c["most"]) / 2
        if c["window"]:
            keys = min(keys, c["window"])
        es = DTYPES[c["cache"]].itemsize
        kv = 2 * keys * c["kv_heads"] * c["head_dim"] * es + 4 * keys / c["page"]
        return {"bytes": c["seqs"] * (kv + 8 * c["heads"] * c["head_dim"] + 4),
                "flops": 4.0 * c["seqs"] * keys * c["heads"] * c["head_dim"]}
    return {"bytes": c["rows"] * (4 * c["vocab"] + 12 + 8 * c["top"]),
            "flops": 5.0 * c["rows"] * c["vocab"]}


# -------------------------------------------------------------------- exact
def _slots_exact(c, seed):
    past, count, table, ring, ends = (t.tolist() for t in _slots_inputs(c, seed))
    ps, pages, width = c["page"], len(ring), len(table[0])
    first, last = ends
    free = ring[:]
    offsets, lengths, positions, slots, failed = [0], [], [], [], 0
    full = False  # the pages have run out: what comes later and wants any has none
    for s, (a, n) in enumerate(zip(past, count)):
        if a < 0 or n < 0:
            if a >= 0:
                for p in table[s][:min(-(-a // ps), width)]:
                    ring[last % pages] = p
                    last += 1
            lengths.append(-1)
            offsets.append(offsets[-1])
            continue
        have, need = -(-a // ps), -(-(a + n) // ps)
        offsets.append(offsets[-1] + n)
        ok = need <= width and offsets[-1] <= c["rows"]
        if ok and need > have:
            full = full or need - have > ends[1] - first
            ok = not full
        if ok:
            for j in range(have, need):
                table[s][j] = free[first % pages]
                first += 1
        else:
            failed += 1
        lengths.append(a + n if ok else a)
        for p in range(a, a + n):
            if len(positions) < c["rows"]:
                positions.append(p)
                e = table[s][p // ps] if ok else -1
                slots.append(e * ps + p % ps if e >= 0 else -1)
    pad = [-1] * (c["rows"] - len(positions))

    def t(a, dtype=torch.int32):
        return torch.tensor(a, dtype=dtype, device="cuda")

    return {"table": t(table), "ring": t(ring), "ends": t([first, last], torch.int64),
            "offsets": t(offsets), "lengths": t(lengths), "positions": t(positions + pad),
            "slots": t(slots + pad), "failed": t([failed])}


def _rope_exact(c, seed):
    qkv, qn, kn, positions, slots, pk, pv = _rope_inputs(c, seed)
    n, hs, kv, hd, d = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["dims"]
    freq, scale = _freqs(c)
    q, k, v = qkv.double().view(n, -1, hd).split((hs, kv, kv), 1)
    if c["norm"]:
        q, k = (t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
                for t, w in ((q, qn), (k, kn)))
    # each pair is a complex number times scale * e^(i angle)
    e = scale * torch.exp(1j * (positions.double()[:, None] * freq.double()))[:, None]

    def turn(t):
        r = t[..., :d]
        z = r.unflatten(-1, (-1, 2)) if c["interleaved"] else r.unflatten(-1, (2, -1)).mT
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * e)
        r = z.flatten(-2) if c["interleaved"] else z.mT.flatten(-2)
        return torch.cat((r, t[..., d:]), -1)

    out = []
    for pool, new in ((pk, turn(k)), (pv, v)):
        pool = pool.double()
        pool.view(-1, kv, hd).index_copy_(0, slots.long(), new)
        out.append(pool)
    return {"q": turn(q), "k": out[0], "v": out[1]}


def _attention_exact(c, seed):
    q, k, v, table, lengths, sinks = _attention_inputs(c, seed)
    kv, hd, ps, group = c["kv_heads"], c["head_dim"], c["page"], c["heads"] // c["kv_heads"]
    y = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for s, n in enumerate(lengths.tolist()):
        j = torch.arange(max(0, n - c["window"]) if c["window"] else 0, n, device="cuda")
        page, at = table[s].long()[j // ps], j % ps
        for g in range(kv):
            kk, vv = k[page, at, g].double(), v[page, at, g].double()
            for h in range(g * group, (g + 1) * group):
                x = (kk * q[s, h].double()).sum(1) / math.sqrt(hd)
                if sinks is not None:
                    x = torch.cat((x, sinks[h:h + 1].double()))
                p = torch.softmax(x, 0)[:len(j)]
                y[s, h] = (p[:, None] * vv).sum(0)
    return y


def _logprobs_exact(c, seed):
    x, ids = _logprobs_inputs(c, seed)
    out = {"logprobs": [], "entropy": [], "top_ids": [], "top_logprobs": []}
    for i in range(0, c["rows"], 64):
        d = x[i:i + 64].double()
        lp = d - torch.logsumexp(d, 1, keepdim=True)
        out["logprobs"].append(lp.gather(1, ids[i:i + 64].long()[:, None])[:, 0])
        out["entropy"].append(-(lp.exp() * lp).sum(1))
        # every candidate of the largest values, ties by the lower index
        rows_ids, rows_lp = [], []
        for r in range(len(d)):
            least = torch.topk(d[r], c["top"]).values[-1]
            at = (d[r] >= least).nonzero()[:, 0]
            at = at[torch.sort(d[r][at], descending=True, stable=True).indices][:c["top"]]
            rows_ids.append(at.int())
            rows_lp.append(lp[r][at])
        out["top_ids"].append(torch.stack(rows_ids))
        out["top_logprobs"].append(torch.stack(rows_lp))
    return {k: torch.cat(v) for k, v in out.items()}


def exact(case, seed):
    return {"slots": _slots_exact, "rope": _rope_exact, "attention": _attention_exact,
            "logprobs": _logprobs_exact}[case["kind"]](case, seed)

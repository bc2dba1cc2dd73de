"""The measured work of a serving step over an 8-bit paged cache, with a prompt that
many sequences share and a draw for every row, through the C-ABI entry points of
infer_hip.

Five kinds of case:

- store: the new rows' keys and values (head norms, rotary positions) quantized as
  they are written into 8-bit pages (a scale for each head of a token), and the same
  tokens read back, as the attention of a prompt's chunk takes them;
- read: whole histories read back from 8-bit pages;
- attention: one new token of each sequence over its 8-bit pages;
- shared: one new token of each sequence, where groups of sequences have a long
  prefix in common that is read once for all of a group;
- sample: a draw for each row of logits, with settings and a random number of its own.

The plain forms are elementary torch operations in 32 bits; in 64 where a value is
rounded to 8 bits or a draw falls next to a border.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step's rows of 64 chats into the cache (32 + 4 heads of 128)
        dict(name="store-decode", kind="store", seqs=64, most=4096, new=1, heads=32, kv_heads=4,
             head_dim=128, norm=True, page=16, out="f16"),
        # a batch of prompt chunks, ragged heads, odd lengths (64 + 8 heads of 64)
        dict(name="store-prompts", kind="store", seqs=9, most=9000, new=889, heads=64, kv_heads=8,
             head_dim=64, norm=False, page=32, out="f32"),
        # one chat's history for its next chunk's attention
        dict(name="read-chat", kind="read", seqs=1, least=1151, most=1151, kv_heads=4, head_dim=128,
             page=16, out="f16"),
        # ragged histories of a batch, in single
        dict(name="read-batch", kind="read", seqs=48, least=1, most=8200, kv_heads=8, head_dim=128,
             page=24, out="f32"),
        # one chat after a 1151-token context: latency
        dict(name="attention-one", kind="attention", seqs=1, least=1152, most=1152, heads=32, kv_heads=4,
             head_dim=128, window=0, sinks=False, page=16),
        # a serving batch of ragged lengths
        dict(name="attention-batch", kind="attention", seqs=64, least=100, most=16384, heads=16, kv_heads=8,
             head_dim=128, window=0, sinks=False, page=16),
        # chats behind one system prompt, short turns of their own
        dict(name="shared-chats", kind="shared", groups=1, seqs=32, prefix=4096, own=600, heads=32,
             kv_heads=4, head_dim=128, sinks=False, page=16, cache="f16"),
        # many questions about one long document, sinks
        dict(name="shared-document", kind="shared", groups=1, seqs=128, prefix=30011, own=300, heads=64,
             kv_heads=8, head_dim=64, sinks=True, page=32, cache="bf16"),
        # three prompts, their requests beside each other, 8-bit pages, heads of 256
        dict(name="shared-prompts", kind="shared", groups=3, seqs=60, prefix=9001, own=1000, heads=16,
             kv_heads=8, head_dim=256, sinks=False, page=64, cache="q8"),
        # one chat's next token: latency
        dict(name="sample-one", kind="sample", rows=1, vocab=151936, settings="chat"),
        # a decode step's rows, every request with settings of its own
        dict(name="sample-batch", kind="sample", rows=61, vocab=201088, settings="mixed"),
        # a large batch
        dict(name="sample-many", kind="sample", rows=500, vocab=151936, settings="mixed"),
    ]


HEADS = ((32, 4, 128), (16, 8, 128), (64, 8, 64), (8, 2, 256), (16, 8, 256), (14, 2, 64), (16, 2, 512),
         (12, 12, 96), (32, 2, 80), (48, 2, 128))

# (temperature, top_k, top_p, min_p): greedy, the whole vocabulary, and usual chat settings
SETTINGS = {
    "chat": ((0.6, 20, 0.95, 0.0),),
    "plain": ((1.0, 0, 1.0, 0.0),),
    "nucleus": ((1.0, 0, 0.95, 0.0), (0.8, 0, 0.9, 0.0)),
    "min": ((1.0, 0, 1.0, 0.05), (1.5, 0, 1.0, 0.1)),
    "mixed": ((0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (0.7, 20, 0.8, 0.0),
              (1.0, 64, 0.95, 0.0), (0.8, 0, 0.95, 0.05), (1.0, 0, 0.9, 0.0), (0.8, 40, 1.0, 0.0)),
}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("store", "read", "attention", "shared", "sample"), (2, 2, 4, 4, 4))[0]
    page = rng.choice((1, 7, 16, 24, 32, 64, 100, 128, 256))
    if kind == "sample":
        vocab = rng.choice((151936, 201088, 248320, 262144, _log(rng, 500, 200000)))
        return dict(kind=kind, rows=_log(rng, 1, max(2, min(500, 70000000 // vocab))), vocab=vocab,
                    settings=rng.choice(("mixed", "mixed", "chat", "plain", "nucleus", "min")))
    heads, kv, hd = rng.choice(HEADS)
    if kind == "store":
        new = rng.choice((1, _log(rng, 2, 900)))
        seqs = _log(rng, 1, max(2, min(500, 25000000 // ((heads + 4 * kv) * hd * new))))
        return dict(kind=kind, seqs=seqs, most=_log(rng, new + 64, 32768), new=new, heads=heads, kv_heads=kv,
                    head_dim=hd, norm=rng.random() < 0.5, page=page, out=rng.choice(("f16", "f32")))
    if kind == "read":
        seqs = _log(rng, 1, 64)
        most = max(1, min(_log(rng, 16, 32768), 200000000 // (seqs * kv * hd)))
        return dict(kind=kind, seqs=seqs, least=max(1, int(most * rng.choice((0.01, 1.0)))), most=most,
                    kv_heads=kv, head_dim=hd, page=page, out=rng.choice(("f16", "f32")))
    if kind == "attention":
        seqs = _log(rng, 1, 128)
        most = max(1, min(_log(rng, 16, 131072), int(900e6 / (seqs * 2 * kv * hd))))
        windowed = rng.random() < 0.2
        return dict(kind=kind, seqs=seqs, least=max(1, int(most * rng.choice((0.01, 0.3, 1.0)))), most=most,
                    heads=heads, kv_heads=kv, head_dim=hd, window=rng.choice((128, 1000)) if windowed else 0,
                    sinks=rng.random() < 0.3, page=page)
    groups = rng.choice((1, 1, 2, 5))
    seqs = groups * _log(rng, 2, 128 // groups)
    prefix = min(_log(rng, 100, 40000), int(5e9 / (seqs * heads * hd)))
    return dict(kind=kind, groups=groups, seqs=seqs, prefix=prefix, own=_log(rng, 1, 1000), heads=heads,
                kv_heads=kv, head_dim=hd, sinks=rng.random() < 0.3, page=page,
                cache=rng.choice(("f16", "bf16", "f32", "q8", "q8")))


# ------------------------------------------------------------------- prepare
class State:
    pass


def _rand(c, seed):
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 31 * len(c["kind"]))

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def uniform(*shape, dtype=torch.float32):
        return torch.rand(shape, generator=g, device="cuda", dtype=dtype)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").int()

    return ints, normal, uniform, shuffled


def _tables(pages_of, width, order):
    """Block tables [seqs, width] that take the pages of `order` in turn, -1 behind them."""
    first = torch.cumsum(pages_of, 0) - pages_of
    j = torch.arange(width, device="cuda")[None]
    at = (first[:, None] + j).clamp(max=len(order) - 1)
    return torch.where(j < pages_of[:, None], order[at], -1).int().contiguous()


def _pool(c, pages, normal, uniform, cache):
    """(k, v, scales of k, scales of v) of `pages` pages with other tokens in them; 8-bit codes as
    normally distributed values leave them, their heads of different sizes."""
    shape = (pages, c["page"], c["kv_heads"], c["head_dim"])
    if cache != "q8":
        return normal(*shape, dtype=DTYPES[cache]), normal(*shape, dtype=DTYPES[cache]), None, None
    k, v = ((normal(*shape, dtype=torch.bfloat16) * 40).clamp(-127, 127).to(torch.int8) for _ in range(2))
    ks, vs = ((0.5 + uniform(*shape[:3])) / 40 for _ in range(2))
    return k, v, ks, vs


def _store_inputs(c, seed):
    ints, normal, uniform, shuffled = _rand(c, seed)
    n, new, hs, kv, hd, ps = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    # a fused product's rows: q, k and v of a row beside each other
    qkv = normal(n * new, (hs + 2 * kv) * hd)
    qn, kn = (1 + 0.1 * normal(hd), 1 + 0.1 * normal(hd)) if c["norm"] else (None, None)
    past = ints(0, max(0, c["most"] - new), n)
    have = (past + new + ps - 1) // ps
    order = shuffled(int(have.sum()) + 8)
    table = _tables(have, -(-(int(past.max()) + new) // ps), order)
    # the step's plan: the rows' positions and slots, each sequence's first row
    positions = (past[:, None] + torch.arange(new, device="cuda", dtype=torch.int32)).flatten()
    seq = torch.arange(n, device="cuda").repeat_interleave(new)
    slots = table[seq, (positions // ps).long()] * ps + positions % ps
    offsets = torch.arange(0, n * new + 1, new, device="cuda", dtype=torch.int32)
    freq = (1.0 / 1e6 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)).float()
    return (qkv, qn, kn, freq, past, table, positions.int(), slots.int().contiguous(), offsets,
            _pool(c, len(order), normal, uniform, "q8"))


def _read_inputs(c, seed):
    ints, normal, uniform, shuffled = _rand(c, seed)
    # two sequences' lengths add up to the same, so that all seeds read as many rows
    lengths = ints(c["least"], c["most"], c["seqs"])
    lengths[1::2] = c["least"] + c["most"] - lengths[0:c["seqs"] // 2 * 2:2]
    if c["seqs"] % 2:
        lengths[-1] = (c["least"] + c["most"]) // 2
    have = (lengths + c["page"] - 1) // c["page"]
    order = shuffled(int(have.sum()) + 8)
    table = _tables(have, -(-c["most"] // c["page"]), order)
    offsets = torch.zeros(c["seqs"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(lengths, 0)
    return table, offsets, _pool(c, len(order), normal, uniform, "q8")


def _attention_inputs(c, seed):
    ints, normal, uniform, shuffled = _rand(c, seed)
    lengths = ints(c["least"], c["most"], c["seqs"])
    have = (lengths + c["page"] - 1) // c["page"]
    # half as many pages again as the sequences use: other sequences' keys
    used = int(have.sum())
    order = shuffled(used + used // 2 + 1)
    table = _tables(have, -(-c["most"] // c["page"]), order)
    pool = _pool(c, len(order), normal, uniform, "q8")
    return normal(c["seqs"], c["heads"], c["head_dim"]), pool, table, lengths, normal(c["heads"]) if c["sinks"] else None


def _shared_inputs(c, seed):
    ints, normal, uniform, shuffled = _rand(c, seed)
    n, groups, ps = c["seqs"], c["groups"], c["page"]
    # whole pages are shared: the first ones of every table of a group; prompts of different lengths
    shared = ints(max(1, c["prefix"] * 2 // 3), c["prefix"], groups)
    shared[0] = c["prefix"]
    shared = (shared // ps).clamp(min=1) * ps
    members = torch.arange(0, n + 1, n // groups, device="cuda", dtype=torch.int32)
    group = torch.arange(n, device="cuda") // (n // groups)
    lengths = shared[group] + ints(1, c["own"], n)
    first = (shared // ps)[group]
    have = (lengths + ps - 1) // ps
    own_pages = have - first
    used = int(own_pages.sum()) + int((shared // ps).sum())
    order = shuffled(used + 8)
    width = int(have.max())
    j = torch.arange(width, device="cuda")[None]
    start = torch.cumsum(shared // ps, 0) - shared // ps
    mine = int((shared // ps).sum()) + torch.cumsum(own_pages, 0) - own_pages
    at = torch.where(j < first[:, None], start[group][:, None] + j, mine[:, None] + j - first[:, None])
    table = torch.where(j < have[:, None], order[at.clamp(max=len(order) - 1)], -1).int().contiguous()
    pool = _pool(c, len(order), normal, uniform, c["cache"])
    return (normal(n, c["heads"], c["head_dim"]), pool, table, lengths.int().contiguous(), members,
            shared.int().contiguous(), normal(c["heads"]) if c["sinks"] else None)


def _sample_inputs(c, seed):
    ints, _, uniform, _ = _rand(c, seed)
    n, vocab = c["rows"], c["vocab"]
    # log probabilities that fall with the logarithm of the rank, steeply in most rows
    x = uniform(n, vocab).mul_(vocab).add_(1).log_()
    x *= -(1.1 + 2.4 * uniform(n, 1))
    x += 18
    presets = torch.tensor(SETTINGS[c["settings"]], dtype=torch.float64, device="cuda")
    picked = presets[ints(0, len(presets) - 1, n).long()]
    # ihip_sampling: temperature, top_k (int32, then 4 bytes of 0), top_p, min_p, seed
    settings = torch.zeros(n, 5, dtype=torch.float64, device="cuda")
    settings[:, 0], settings[:, 2], settings[:, 3] = picked[:, 0], picked[:, 2], picked[:, 3]
    settings.view(torch.int64)[:, 1] = picked[:, 1].long()
    return x, settings, uniform(n, dtype=torch.float64)


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


def _pages(H, k, v, ks, vs):
    code = {torch.float32: H.F32, torch.float16: H.F16, torch.bfloat16: H.BF16, torch.int8: H.Q8_HEAD}
    scales = dict(k_scale=ks.data_ptr(), v_scale=vs.data_ptr()) if ks is not None else {}
    return H.Pages(k=k.data_ptr(), v=v.data_ptr(), pages=k.shape[0], page_size=k.shape[1],
                   kv_heads=k.shape[2], head_dim=k.shape[3], dtype=code[k.dtype], **scales)


def prepare(case, seed):
    c, s = case, State()
    s.case = c
    kind = c["kind"]
    if kind == "store":
        (s.qkv, s.qn, s.kn, s.freq, s.past, s.table, s.positions, s.slots, s.offsets,
         s.pool) = _store_inputs(c, seed)
        s.q = torch.zeros((len(s.slots), c["heads"], c["head_dim"]), device="cuda")
    elif kind == "read":
        s.table, s.offsets, s.pool = _read_inputs(c, seed)
        s.rows = int(s.offsets[-1])
    elif kind == "attention":
        s.q, s.pool, s.table, s.lengths, s.sinks = _attention_inputs(c, seed)
        s.y = torch.zeros_like(s.q)
    elif kind == "shared":
        s.q, s.pool, s.table, s.lengths, s.members, s.shared, s.sinks = _shared_inputs(c, seed)
        s.y = torch.zeros_like(s.q)
    else:
        s.x, s.settings, s.u = _sample_inputs(c, seed)
        s.ids = torch.zeros(c["rows"], dtype=torch.int32, device="cuda")
        s.probs = torch.zeros(c["rows"], device="cuda")
    if kind in ("store", "read"):
        rows = len(s.slots) if kind == "store" else s.rows
        s.k, s.v = (torch.zeros((rows, c["kv_heads"], c["head_dim"]), dtype=DTYPES[c["out"]], device="cuda")
                    for _ in range(2))
    if own:
        H, s.ctx = _ctx()
        s.h = H
        if kind != "sample":
            s.pages = _pages(H, *s.pool)
        if kind == "store":
            s.rope = H.Rope(freq=s.freq.data_ptr(), dims=c["head_dim"], scale=1.0)
        if kind in ("store", "read"):
            s.out = {"f16": H.F16, "f32": H.F32}[c["out"]]
    torch.cuda.synchronize()
    return s


# ----------------------------------------------------------------- one pass
def _quantize(x):
    """Codes and scales of heads: the scale is 1 / 127 of the largest magnitude, in single."""
    scale = (x.abs().amax(-1) / 127).float()
    codes = torch.where(scale[..., None] > 0, torch.round(x / scale[..., None].double()), 0.0)
    return codes.clamp(-127, 127).to(torch.int8), scale


def _read_back(s, table, first, offsets, rows):
    c = s.case
    k, v, ks, vs = s.pool
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(offsets[1:].long(), r, right=True)
    pos = r - offsets[seq] + (first[seq] if first is not None else 0)
    page, at = table[seq, pos // c["page"]].long(), pos % c["page"]
    s.k.copy_(k[page, at].float() * ks[page, at][..., None])
    s.v.copy_(v[page, at].float() * vs[page, at][..., None])


def _store_plain(s):
    c = s.case
    n, hs, kv, hd = len(s.slots), c["heads"], c["kv_heads"], c["head_dim"]
    x = s.qkv.view(n, hs + 2 * kv, hd)
    # (in 64 bits: what is next to the border of two codes)
    q, k, v = x[:, :hs].double(), x[:, hs:hs + kv].double(), x[:, hs + kv:].double()
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s.qn.double()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s.kn.double()
    angle = s.positions.double()[:, None] * s.freq.double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(t):
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    s.q.copy_(turn(q))
    at = s.slots.long()
    for pool, scales, new in ((s.pool[0], s.pool[2], turn(k)), (s.pool[1], s.pool[3], v)):
        codes, scale = _quantize(new)
        pool.view(-1, kv, hd)[at] = codes
        scales.view(-1, kv)[at] = scale
    _read_back(s, s.table, s.past, s.offsets, n)
    return {"q": s.q, "k": s.k, "v": s.v}


def _read_plain(s):
    _read_back(s, s.table, None, s.offsets, s.rows)
    return {"k": s.k, "v": s.v}


def _gathered(pool, table):
    """(keys, values) [n, width * page, kv, hd] in single of tables [n, width]."""
    t = table.long().clamp(min=0)
    out = []
    for x, scale in ((pool[0], pool[2]), (pool[1], pool[3])):
        g = x[t].float()
        if scale is not None:
            g = g * scale[t][..., None]
        out.append(g.flatten(1, 2))
    return out


def _attention_plain(s):
    c = s.case
    n, hs, kv, hd, ps = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    width = s.table.shape[1]
    # sequences in groups whose gathered keys stay small
    step = max(1, int(2e9 / (width * ps * kv * hd * 4)))
    for i in range(0, n, step):
        ln = s.lengths[i:i + step].long()
        m = len(ln)
        k, v = _gathered(s.pool, s.table[i:i + step])
        q = s.q[i:i + step].view(m, kv, hs // kv, hd) * hd ** -0.5
        x = q @ k.permute(0, 2, 3, 1).contiguous()
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
        s.y[i:i + step] = (p @ v.permute(0, 2, 1, 3).contiguous() / total).view(m, hs, hd)
    return s.y


def _shared_plain(s):
    c = s.case
    hs, kv, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    m = c["seqs"] // c["groups"]
    group = hs // kv
    for g, common in enumerate((s.shared // ps).tolist()):
        lo, hi = g * m, (g + 1) * m
        q = s.q[lo:hi].view(m, kv, group, hd) * hd ** -0.5
        # the prefix: all members' queries of a KV head against keys that are gathered once
        k, v = _gathered(s.pool, s.table[lo:lo + 1, :common])
        qa = q.transpose(0, 1).reshape(kv, m * group, hd)
        xa = (qa @ k[0].permute(1, 2, 0).contiguous()).view(kv, m, group, -1).transpose(0, 1)
        # the members' own tokens
        kb, vb = _gathered(s.pool, s.table[lo:hi, common:])
        xb = q @ kb.permute(0, 2, 3, 1).contiguous()
        j = torch.arange(xb.shape[-1], device="cuda")[None] + common * ps
        xb = xb.masked_fill((j >= s.lengths[lo:hi, None])[:, None, None], -math.inf)
        top = torch.maximum(xa.amax(-1, keepdim=True), xb.amax(-1, keepdim=True))
        if c["sinks"]:
            sink = s.sinks.view(1, kv, group, 1)
            top = torch.maximum(top, sink)
        pa, pb = torch.exp(xa - top), torch.exp(xb - top)
        total = pa.sum(-1, keepdim=True) + pb.sum(-1, keepdim=True)
        if c["sinks"]:
            total = total + torch.exp(sink - top)
        y = pa.transpose(0, 1).reshape(kv, m * group, -1) @ v[0].transpose(0, 1).contiguous()
        y = y.view(kv, m, group, hd).transpose(0, 1) + pb @ vb.permute(0, 2, 1, 3).contiguous()
        s.y[lo:hi] = (y / total).reshape(m, hs, hd)
    return s.y


def _sample_plain(s):
    c = s.case
    for i in range(0, c["rows"], 64):
        x, u = s.x[i:i + 64].double(), s.u[i:i + 64, None]
        temp, top_p, min_p = (s.settings[i:i + 64, j:j + 1] for j in (0, 2, 3))
        top_k = s.settings[i:i + 64].view(torch.int64)[:, 1:2]
        # (64 bits: a draw is a comparison of running sums)
        w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(temp > 0, temp, 1.0))
        # the filters' order: the largest logit first, the lowest id on a tie
        sx, order = torch.sort(x, dim=1, descending=True, stable=True)
        sw = w.gather(1, order)
        kth = sx.gather(1, (top_k - 1).clamp(0, c["vocab"] - 1))
        keep = torch.where(top_k > 0, sx >= kth, True)
        sw = torch.where(keep, sw, 0.0)
        before = torch.cumsum(sw, 1) - sw
        keep &= (top_p >= 1) | (before < top_p * sw.sum(1, keepdim=True))
        keep &= (min_p <= 0) | (sw >= min_p * sw[:, :1])
        sw = torch.where(keep, sw, 0.0)
        # without a filter the draw goes by id
        free = (top_k == 0) & (top_p >= 1) & (min_p <= 0)
        p = torch.where(free, w, sw)
        run = torch.cumsum(p, 1)
        at = ((run <= u * run[:, -1:]) | (p <= 0)).int().argmin(1, keepdim=True)
        ids = torch.where(free, at, order.gather(1, at))
        ids = torch.where(temp > 0, ids, order[:, :1])
        s.ids[i:i + 64] = ids[:, 0].int()
        s.probs[i:i + 64] = torch.where(temp > 0, p.gather(1, at) / run[:, -1:], 1.0)[:, 0].float()
    return {"ids": s.ids, "probs": s.probs}


def run(s):
    c = s.case
    kind = c["kind"]
    if not own:
        return {"store": _store_plain, "read": _read_plain, "attention": _attention_plain,
                "shared": _shared_plain, "sample": _sample_plain}[kind](s)
    H, h = s.h, s.ctx.h
    L = H.lib()
    if kind == "store":
        hs, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
        q, stride, rows = s.qkv.data_ptr(), (hs + 2 * kv) * hd, len(s.slots)
        H.check(L.ihip_enqueue_paged_qkrope(
            h, q, stride, q + 4 * hs * hd, stride, q + 4 * (hs + kv) * hd, stride, rows, hs,
            s.qn.data_ptr() if c["norm"] else 0, s.kn.data_ptr() if c["norm"] else 0, 1e-6,
            H.C.byref(s.rope), s.positions.data_ptr(), s.slots.data_ptr(), H.C.byref(s.pages),
            s.q.data_ptr()), "qkrope")
        H.check(L.ihip_enqueue_paged_read(
            h, H.C.byref(s.pages), s.table.data_ptr(), s.table.shape[1], s.past.data_ptr(),
            s.offsets.data_ptr(), c["seqs"], rows, s.out, s.k.data_ptr(), s.v.data_ptr()), "read")
        return {"q": s.q, "k": s.k, "v": s.v}
    if kind == "read":
        H.check(L.ihip_enqueue_paged_read(
            h, H.C.byref(s.pages), s.table.data_ptr(), s.table.shape[1], 0, s.offsets.data_ptr(),
            c["seqs"], s.rows, s.out, s.k.data_ptr(), s.v.data_ptr()), "read")
        return {"k": s.k, "v": s.v}
    if kind == "attention":
        H.check(L.ihip_enqueue_paged_attention(
            h, s.q.data_ptr(), 0, H.C.byref(s.pages), s.table.data_ptr(), s.table.shape[1],
            s.lengths.data_ptr(), s.y.data_ptr(), c["seqs"], c["heads"], c["window"],
            s.sinks.data_ptr() if c["sinks"] else 0, 0.0), "attention")
        return s.y
    if kind == "shared":
        H.check(L.ihip_enqueue_paged_attention_shared(
            h, s.q.data_ptr(), 0, H.C.byref(s.pages), s.table.data_ptr(), s.table.shape[1],
            s.lengths.data_ptr(), 0, c["seqs"], s.members.data_ptr(), s.shared.data_ptr(), c["groups"],
            s.y.data_ptr(), c["seqs"], c["heads"], 0, s.sinks.data_ptr() if c["sinks"] else 0, 0.0), "shared")
        return s.y
    H.check(L.ihip_enqueue_sample_rows(
        h, s.x.data_ptr(), c["rows"], c["vocab"], 0, s.settings.data_ptr(), s.u.data_ptr(),
        s.ids.data_ptr(), s.probs.data_ptr()), "sample")
    return {"ids": s.ids, "probs": s.probs}


# --------------------------------------------------------------------- work
def work(case):
    c = case
    kind = c["kind"]
    if kind == "sample":
        return {"bytes": c["rows"] * (4 * c["vocab"] + 56), "flops": 6.0 * c["rows"] * c["vocab"]}
    kv, hd = c["kv_heads"], c["head_dim"]
    es = DTYPES[c["out"]].itemsize if "out" in c else 0
    token = 2 * kv * (hd + 4)  # of the 8-bit pages
    if kind == "store":
        rows, qw, kw = c["seqs"] * c["new"], c["heads"] * hd, kv * hd
        # q in and out; k and v in, into the pages, out of them, and out
        return {"bytes": rows * (8 * qw + 8 * kw + 2 * token + 2 * es * kw + 8),
                "flops": rows * (qw + kw) * (6.0 if c["norm"] else 3.0) + 6.0 * rows * kw}
    if kind == "read":
        rows = c["seqs"] * (c["least"] + c["most"]) // 2
        return {"bytes": rows * (token + 2 * es * kv * hd), "flops": 2.0 * rows * kv * hd}
    if kind == "attention":
        # (the mean length: a case's own lengths follow the seed)
        keys = (c["least"] + c["most"]) / 2
        if c["window"]:
            keys = min(keys, c["window"])
        return {"bytes": c["seqs"] * (keys * token + 4 * keys / c["page"] + 8 * c["heads"] * hd + 4),
                "flops": 4.0 * c["seqs"] * keys * c["heads"] * hd}
    if c["cache"] != "q8":
        token = 2 * kv * hd * DTYPES[c["cache"]].itemsize
    # the first group's prefix whole, the others' between two thirds of it and that
    prefix = c["prefix"] * (1 + (c["groups"] - 1) * 5 / 6) / c["groups"]
    mine = (1 + c["own"]) / 2
    return {"bytes": c["groups"] * prefix * token + c["seqs"] * (mine * token + 8 * c["heads"] * hd + 4),
            "flops": 4.0 * c["seqs"] * (prefix + mine) * c["heads"] * hd}


# -------------------------------------------------------------------- exact
def _store_exact(c, seed):
    qkv, qn, kn, freq, _, _, positions, _, _, _ = _store_inputs(c, seed)
    n, hs, kv, hd = len(positions), c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = qkv.double().view(n, -1, hd).split((hs, kv, kv), 1)
    if c["norm"]:
        q, k = (t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
                for t, w in ((q, qn), (k, kn)))
    # each pair is a complex number times e^(i angle)
    e = torch.exp(1j * (positions.double()[:, None] * freq.double()))[:, None]

    def turn(t):
        z = torch.view_as_complex(t.unflatten(-1, (2, -1)).mT.contiguous()) * e
        return torch.view_as_real(z).mT.flatten(-2)

    def stored(t):
        d = (t.abs().max(-1, keepdim=True).values / 127).float().double()
        return (t / d).round() * d

    return {"q": turn(q), "k": stored(turn(k)), "v": stored(v)}


def _read_exact(c, seed):
    table, offsets, (k, v, ks, vs) = _read_inputs(c, seed)
    out = []
    for codes, scale in ((k, ks), (v, vs)):
        rows = []
        for s in range(c["seqs"]):
            n = int(offsets[s + 1] - offsets[s])
            j = torch.arange(n, device="cuda")
            page, at = table[s].long()[j // c["page"]], j % c["page"]
            rows.append(codes[page, at].double() * scale[page, at].double()[..., None])
        out.append(torch.cat(rows))
    return {"k": out[0], "v": out[1]}


def _one_sequence(q, pool, row, length, window, ps, group, sinks):
    """One token's attention over a sequence in 64 bits; q [heads, hd]."""
    y = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    j = torch.arange(max(0, length - window) if window else 0, length, device="cuda")
    page, at = row.long()[j // ps], j % ps
    for g in range(q.shape[0] // group):
        kk, vv = pool[0][page, at, g].double(), pool[1][page, at, g].double()
        if pool[2] is not None:
            kk, vv = kk * pool[2][page, at, g].double()[:, None], vv * pool[3][page, at, g].double()[:, None]
        hs = slice(g * group, (g + 1) * group)
        x = kk @ q[hs].double().t().contiguous() / math.sqrt(q.shape[1])
        if sinks is not None:
            x = torch.cat((x, sinks[None, hs].double()))
        p = torch.softmax(x, 0)[:len(j)]
        y[hs] = p.t().contiguous() @ vv
    return y


def _attention_exact(c, seed):
    q, pool, table, lengths, sinks = _attention_inputs(c, seed)
    return torch.stack([_one_sequence(q[s], pool, table[s], n, c["window"], c["page"],
                                      c["heads"] // c["kv_heads"], sinks)
                        for s, n in enumerate(lengths.tolist())])


def _shared_exact(c, seed):
    # every sequence by itself, over its own table
    q, pool, table, lengths, _, _, sinks = _shared_inputs(c, seed)
    return torch.stack([_one_sequence(q[s], pool, table[s], n, 0, c["page"], c["heads"] // c["kv_heads"], sinks)
                        for s, n in enumerate(lengths.tolist())])


def _sample_exact(c, seed):
    x, settings, u = _sample_inputs(c, seed)
    ids, probs = [], []
    for r in range(c["rows"]):
        (t, _, top_p, min_p, _), k = settings[r].tolist(), int(settings[r].view(torch.int64)[1])
        row = x[r]
        best = int((row == row.max()).nonzero()[0])
        if t <= 0:
            ids.append(best)
            probs.append(1.0)
            continue
        p = torch.softmax(row.double() / t, 0)
        if k == 0 and top_p >= 1 and min_p <= 0:
            at = torch.arange(c["vocab"], device="cuda")
        else:
            least = -math.inf if k == 0 else float(torch.topk(row, min(k, c["vocab"])).values[-1])
            at = (row >= least).nonzero()[:, 0]
            at = at[torch.sort(-row[at], stable=True).indices]
            if top_p < 1:
                run = torch.cumsum(p[at], 0)
                mass = run[-1] if k > 0 else 1.0
                at = at[:int((run < top_p * mass).sum()) + 1]
            if min_p > 0:
                at = at[p[at] >= min_p * p[at[0]]]
        run = torch.cumsum(p[at], 0)
        i = min(int((run <= u[r] * run[-1]).sum()), len(at) - 1)
        ids.append(int(at[i]))
        probs.append(float(p[at[i]] / run[-1]))
    return {"ids": torch.tensor(ids, dtype=torch.int32, device="cuda"),
            "probs": torch.tensor(probs, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    return {"store": _store_exact, "read": _read_exact, "attention": _attention_exact,
            "shared": _shared_exact, "sample": _sample_exact}[case["kind"]](case, seed)

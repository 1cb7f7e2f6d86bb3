"""Operators of beam search over long contexts, as measurable cases.

What one such program runs between the projections of the 2B decoder and for its next set of beams (8 query / 2 kv
heads of 256, 18 DeltaNet layers with states of 16 heads, vocabulary 248320):

  attention  `q35.attention_core_paged` over a pool of `q35.Q4` pages: q/k norms, rotary, append of the new tokens'
             keys and values in 4 bits, causal attention over the cache, sigmoid gate; and `q35.pages_read`, what the
             cache holds of the new tokens (the value that each code stands for)
  select     `q35.beam_select`: the highest of all continuations of each group's beams
  reorder    `q35.states_fork`: the states of the sequences that go on, in place

A cached row of 256 values: 8 groups of 32, each with a scale s (an f16 of 7 significant bits) and a zero z (0..15) in
one 16-bit word; the value of code c is s (c - z).  Row: 128 bytes of codes (value d in nibble d % 2 of byte d / 2), 8 words.

`own` false computes them with elementary torch operations, true with the framework's kernels.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
HEAD_DIM, ROT, EPS, THETA = 256, 64, 1e-6, 1e7
VOCAB = 248320
ROW = HEAD_DIM // 2 + HEAD_DIM // 16  # bytes of a cached row
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _q35():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-3.5_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q35
    return q35


# ---------------------------------------------------------------- cases

def _att(name, page, seqs, n, ctx, spread=1, heads=8, kv_heads=2, mix=0):
    c = dict(op="attention", page=page, seqs=seqs, n=n, ctx=ctx, spread=spread, heads=heads, kv_heads=kv_heads, mix=mix)
    return dict(name=name, **c) if name else c


def _sel(name, dtype, groups, beams, k, vocab=VOCAB, masked=0, ended=0, first=False, mix=0):
    c = dict(op="select", dtype=dtype, groups=groups, beams=beams, k=k, vocab=vocab, masked=masked, ended=ended, first=first, mix=mix)
    return dict(name=name, **c) if name else c


def _ord(name, rows, beams, layers, heads, moved=0.6, mix=0):
    c = dict(op="reorder", rows=rows, beams=beams, layers=layers, heads=heads, moved=moved, mix=mix)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one user's next token in a short conversation: latency
        _att("q4_token", 64, 1, 1, 517),
        # 8 beams of one long document, 5 users: the cache's stream, from the caches of the card
        _att("q4_beams", 64, 40, 1, 4096, spread=2, mix=1),
        # 33 users' next tokens, contexts of 8192 to 32768 tokens: the cache's stream
        _att("q4_serve", 32, 33, 1, 32768, spread=4, mix=2),
        # 12 sequences whose 5 drafted tokens are checked
        _att("q4_drafts", 16, 12, 5, 8191, spread=3, mix=3),
        # one long prompt's next chunk behind what is cached already
        _att("q4_chunk", 64, 1, 2048, 14336),
        # 4 beams of one user, twice as many candidates (so that ended ones leave enough): latency
        _sel("select_one", "f32", 1, 4, 8),
        # 32 users of 8 beams, some of them ended
        _sel("select_serve", "f32", 32, 8, 16, ended=20, mix=1),
        # 10 users of 5 beams, 16-bit logits over a smaller vocabulary of odd size, a part of it masked off
        _sel("select_masked", "bf16", 10, 5, 5, vocab=50257, masked=999, mix=2),
        # the first step of 16 users: only their first beams are live
        _sel("select_first", "f16", 16, 8, 8, first=True, mix=3),
        # 4 beams of a 4-layer decoder of 4 heads
        _ord("reorder_small", 4, 4, 3, 4, mix=4),
        # 8 beams of the 2B decoder
        _ord("reorder_beams", 8, 8, 18, 16, mix=5),
        # 9 users of 7 beams
        _ord("reorder_serve", 63, 7, 18, 16, mix=6),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "select", "select", "reorder"])
    mix = rng.randint(0, 10 ** 6)
    if op == "attention":
        heads, kv = rng.choice([(8, 2), (8, 2), (8, 2), (4, 1), (6, 2), (4, 4), (8, 1), (16, 2)])
        page = rng.choice([16, 32, 64, 128])
        kind = rng.choice(["tokens", "tokens", "drafts", "chunk"])
        if kind == "tokens":
            return _att(None, page, _log(rng, 1, 64), 1, _log(rng, 1, 16000), rng.randint(1, 4), heads, kv, mix)
        if kind == "drafts":
            return _att(None, page, _log(rng, 1, 20), rng.randint(2, 9), _log(rng, 1, 9000), rng.randint(1, 4), heads, kv, mix)
        return _att(None, page, rng.randint(1, 3), _log(rng, 10, 700), rng.choice([0, _log(rng, 1, 6000)]), rng.randint(1, 3), heads,
                    kv, mix)
    if op == "select":
        groups, beams = _log(rng, 1, 30), _log(rng, 1, 12)
        vocab = rng.choice([VOCAB, _log(rng, 100, 200000)])
        if groups * beams * vocab > 60 * 10 ** 6:
            groups = max(1, 60 * 10 ** 6 // (beams * vocab))
        return _sel(None, rng.choice(["f32", "f16", "bf16"]), groups, beams, rng.randint(1, 2 * beams), vocab,
                    rng.choice([0, rng.randint(1, vocab // 3)]), rng.choice([0, rng.randint(1, groups * beams)]), rng.random() < 0.2, mix)
    beams = _log(rng, 2, 12)
    return _ord(None, beams * _log(rng, 1, 40 // beams), beams, rng.choice([3, 6, 18]), rng.choice([4, 16]), rng.uniform(0.1, 1.0), mix)


def _contexts(case):
    """Tokens cached before, of every sequence."""
    r = random.Random(case["mix"])
    lo = max(1, case["ctx"] // case["spread"])
    return [case["ctx"] if i == 0 or case["ctx"] == 0 else r.randint(lo, case["ctx"]) for i in range(case["seqs"])]


def _parents(case):
    """Row j goes on from a row of its own group; some rows end (-1)."""
    r = random.Random(case["mix"])
    p = []
    for j in range(case["rows"]):
        g = j // case["beams"] * case["beams"]
        p.append(g + r.randrange(case["beams"]) if r.random() < case["moved"] else j)
    if len(p) > 5:
        p[r.randrange(len(p))] = -1
    return p


# ---------------------------------------------------------------- a cached row

def _pack(y):
    """Rows y [..., 256] (f32) as the cache holds them: uint8 [..., 144]."""
    lead = y.shape[:-1]
    g = y.reshape(*lead, HEAD_DIM // 32, 32)
    fine = g.isfinite().all(-1)
    g = torch.where(fine[..., None], g, 0.0).double().clamp(-32768.0, 32768.0)
    lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    step = (hi - lo) / 15.0
    # the smallest f16 of 7 significant bits that is not below it
    bits = step.float().half().view(torch.int16).int() & ~15
    bits = bits + 16 * (bits.short().view(torch.float16).double() < step).int()
    s = bits.short().view(torch.float16).double()
    some = s > 0
    div = torch.where(some, s, 1.0)
    z = torch.where(some, (-lo / div).round(), 0.0)
    c = torch.where(some[..., None], ((g / div[..., None]).round() + z[..., None]).clamp(0.0, 15.0), 0.0)
    c = torch.where(fine[..., None], c, 0.0).to(torch.uint8).reshape(*lead, HEAD_DIM // 2, 2)
    word = torch.where(fine, bits | z.int(), 0x7FF0).short()
    return torch.cat([c[..., 0] | (c[..., 1] << 4), word.view(torch.uint8)], -1)


def _unpack(rows):
    """The values (f32; each is an f16) of cached rows uint8 [..., 144]."""
    lead = rows.shape[:-1]
    codes, word = rows[..., :HEAD_DIM // 2], rows[..., HEAD_DIM // 2:].contiguous().view(torch.int16)
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*lead, HEAD_DIM // 32, 32).float()
    s, z = (word & ~15).view(torch.float16).float(), (word & 15).float()
    return (s[..., None] * (c - z[..., None])).reshape(*lead, HEAD_DIM)


# ---------------------------------------------------------------- inputs

def _pool(g, case, pages):
    """[1][pages][2][kv heads][page][144]: keys and values of unit size."""
    shape = (pages, 2, case["kv_heads"], case["page"])
    data = torch.empty((1, *shape, ROW), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 17) // (2 * case["kv_heads"] * case["page"]))
    for p0 in range(0, pages, step):
        part = data[0, p0:p0 + step]
        part.copy_(_pack(torch.randn((*part.shape[:-1], HEAD_DIM), generator=g, device=DEV)))
    return data


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cpu = torch.Generator()
    cpu.manual_seed(seed)
    s = {"case": case}

    def normal(*shape, sigma=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=DEV) * sigma + mean

    if case["op"] == "attention":
        ctx, n, page, B = _contexts(case), case["n"], case["page"], case["seqs"]
        need = [-(-(c + n) // page) for c in ctx]
        pages = sum(need) + 3
        ids = torch.randperm(pages, generator=cpu).tolist()
        width = max(need) + 1
        table, at = [], 0
        for k in need:
            table.append(ids[at:at + k] + [-1] * (width - k))
            at += k
        T, H, KV, longest = B * n, case["heads"], case["kv_heads"], max(ctx) + n
        ang = torch.arange(longest, dtype=torch.float64)[:, None] * (
            THETA ** (-torch.arange(0, ROT, 2, dtype=torch.float64) / ROT))[None, :]
        ang = torch.cat([ang, ang], 1)
        new = [c + i for c in ctx for i in range(n)]
        s.update(data=_pool(g, case, pages), table=_i32(table), start=_i32([n * b for b in range(B + 1)]), pos=_i32(ctx),
                 qg=normal(T, H * 2 * HEAD_DIM), k=normal(T, KV * HEAD_DIM, sigma=0.7), v=normal(T, KV * HEAD_DIM),
                 qw=normal(HEAD_DIM, sigma=0.2, mean=0.6), kw=normal(HEAD_DIM, sigma=0.2),
                 cos=ang.cos().float().to(DEV), sin=ang.sin().float().to(DEV), longest=longest,
                 rows=_i32([b for b in range(B) for _ in range(n)]), at=_i32(new))
    elif case["op"] == "select":
        R, V = case["groups"] * case["beams"], case["vocab"]
        x = torch.empty((R, V), dtype=DTYPES[case["dtype"]], device=DEV)
        for r0 in range(0, R, 64):
            x[r0:r0 + 64] = normal(min(64, R - r0), V, sigma=2.5)
        if case["masked"]:
            x[:, torch.randperm(V, generator=cpu)[:case["masked"]].to(DEV)] = -math.inf
        score = normal(case["groups"], case["beams"], sigma=1.5, mean=-20.0)
        ended = torch.full((R,), -1, dtype=torch.int32)
        ended[torch.randperm(R, generator=cpu)[:case["ended"]]] = V - 3  # the end's token
        if case["first"]:
            score[:, 1:] = -math.inf
            score[:, 0] = 0.0
            ended[:] = -1
        s.update(x=x, score=score, ended=ended.to(DEV) if case["ended"] else None)
    else:
        B, h = case["rows"], case["heads"]
        states = []
        for _ in range(case["layers"]):
            states += [normal(B, h, 128, 128), normal(B, h * 384, 3)]
        s.update(states=states, parents=_i32(_parents(case)))
    if own:
        q = _q35()
        if case["op"] == "attention":
            s["pool"] = q.PagePool(s["data"])
            s["dims"] = q.make_dims(attn_heads=case["heads"], kv_heads=case["kv_heads"], head_dim=HEAD_DIM, rot_dim=ROT, eps=EPS,
                                    theta=THETA)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        q = _q35()
        if op == "attention":
            out = q.attention_core_paged(s["dims"], s["pool"], 0, s["qg"], s["k"], s["v"], s["start"], s["pos"], s["table"],
                                         s["qw"], s["kw"], s["cos"], s["sin"])
            return {"out": out, "held": q.pages_read(s["pool"], 0, s["table"], s["rows"], s["at"])}
        if op == "select":
            r = q.beam_select(s["x"], s["score"], s["case"]["k"], ended=s["ended"])
            return {"scores": r.scores, "parents": r.parents, "tokens": r.tokens}
        q.states_fork(s["states"], s["parents"])
        return {"states": s["states"]}
    return {"attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder}[op](s)


def _plain_rotate(x, cos, sin):
    a = x[..., :ROT]
    turned = torch.cat([-a[..., ROT // 2:], a[..., :ROT // 2]], -1)
    return torch.cat([a * cos + turned * sin, x[..., ROT:]], -1)


def _plain_attention(s):
    c, pool, page = s["case"], s["data"][0], s["case"]["page"]
    H, KV, B, n = c["heads"], c["kv_heads"], c["seqs"], c["n"]
    rep, T = H // KV, B * n
    rows, at = s["rows"].long(), s["at"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    # keys in 64 bits: what they are rounded to must not hang on the last bit of a sum
    k = s["k"].view(T, KV, HEAD_DIM).double()
    k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * (1.0 + s["kw"].double())
    k = _plain_rotate(k, cos.double(), sin.double()).float()
    pg, slot = s["table"][rows, at // page].long(), at % page
    pool[pg, 0, :, slot] = _pack(k)
    pool[pg, 1, :, slot] = _pack(s["v"].view(T, KV, HEAD_DIM))
    held = _unpack(pool[pg, :, :, slot]).half()
    qg = s["qg"].view(T, H, 2, HEAD_DIM)
    q = qg[:, :, 0]
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * (1.0 + s["qw"])
    q = _plain_rotate(q, cos, sin).view(B, n, KV, rep, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(B * KV, rep * n, HEAD_DIM)
    used = s["table"][:, :-(-s["longest"] // page)].clamp(min=0).long()
    L = used.shape[1] * page
    kv = _unpack(pool[used].permute(2, 0, 3, 1, 4, 5).reshape(2, B * KV, L, ROW))
    p = torch.matmul(q, kv[0].transpose(1, 2).contiguous()).view(B, KV, rep, n, L) * HEAD_DIM ** -0.5
    p = p.masked_fill(torch.arange(L, device=DEV) > at.view(B, 1, 1, n, 1), -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(B * KV, rep * n, L), kv[1]).view(B, KV, rep, n, HEAD_DIM) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(T, H, HEAD_DIM)
    return {"out": (o / (1.0 + (-qg[:, :, 1]).exp())).reshape(T, H * HEAD_DIM), "held": held}


def _plain_select(s):
    c, x = s["case"], s["x"]
    G, W, V, k = c["groups"], c["beams"], c["vocab"], c["k"]
    per = min(k, V)
    score = s["score"].double().view(G * W, 1)
    # one whole number per logit, larger for a larger one and, of equal ones, for the lower token
    bits = (x.float() + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (V - 1 - torch.arange(V, device=DEV))
    ids = V - 1 - (key.topk(per, 1).values & 0xFFFFFFFF)
    # in 64 bits: continuations of different beams lie close together
    d = x.double()
    m = d.amax(1, keepdim=True)
    lse = m + (d - m).exp().sum(1, keepdim=True).log()
    cand = score + (d.gather(1, ids) - lse)
    if s["ended"] is not None:
        over, first = (s["ended"] >= 0)[:, None], torch.arange(per, device=DEV) == 0
        cand = torch.where(over, torch.where(first, score, -math.inf), cand)
        ids = torch.where(over, s["ended"].long()[:, None], ids)
    cand = torch.where(score > -math.inf, cand, -math.inf).view(G, W * per)
    best = cand.sort(dim=1, descending=True, stable=True)
    at, val = best.indices[:, :k], best.values[:, :k]
    none = val == -math.inf
    parents = torch.arange(G, device=DEV)[:, None] * W + at // per
    tokens = ids.view(G, W * per).gather(1, at)
    return {"scores": val.float(), "parents": torch.where(none, -1, parents).int(), "tokens": torch.where(none, -1, tokens).int()}


def _plain_reorder(s):
    p = s["parents"].long()
    src = torch.where(p >= 0, p, torch.arange(p.numel(), device=DEV))
    return {"states": [t.copy_(t[src]) for t in s["states"]]}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "attention":
        H, KV, n, ctx = case["heads"], case["kv_heads"], case["n"], _contexts(case)
        T = n * len(ctx)
        # the cached rows, the new ones (f32 in, 4 bits out, their values), queries, gates and outputs, rotary rows
        moved = 2 * KV * (sum(ctx) * ROW + T * (4 * HEAD_DIM + ROW + 2 * HEAD_DIM)) + T * H * 3 * HEAD_DIM * 4 + T * 2 * ROT * 4
        return {"bytes": moved, "flops": 4 * HEAD_DIM * H * sum(n * c + n * (n + 1) // 2 for c in ctx)}
    if case["op"] == "select":
        rows = case["groups"] if case["first"] else case["groups"] * case["beams"] - case["ended"]
        n = rows * case["vocab"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["groups"] * (8 * case["beams"] + 12 * case["k"]) + 1, "flops": 5 * n}
    p = _parents(case)
    moved = [(j, q) for j, q in enumerate(p) if q >= 0 and q != j]
    row = case["layers"] * case["heads"] * (128 * 128 + 384 * 3) * 4
    return {"bytes": (len(moved) + len({q for _, q in moved})) * row + 4 * len(p), "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reorder":
        src = [j if q < 0 else q for j, q in enumerate(_parents(case))]
        return {"states": [torch.stack([t[q] for q in src]).double() for t in s["states"]]}
    if case["op"] == "select":
        W, k = case["beams"], case["k"]
        over = s["ended"].tolist() if s["ended"] is not None else [-1] * (case["groups"] * W)
        res = {"scores": [], "parents": [], "tokens": []}
        for g in range(case["groups"]):
            c = s["score"][g].double()[:, None] + torch.log_softmax(s["x"][g * W:(g + 1) * W].double(), 1)
            for w in range(W):
                if over[g * W + w] >= 0:
                    c[w] = -math.inf
                    c[w, over[g * W + w]] = s["score"][g, w].double()
            val, at = torch.sort(c.flatten(), descending=True, stable=True)
            val, at = val[:k], at[:k]
            gone = val.isneginf()
            res["scores"].append(val)
            res["parents"].append(torch.where(gone, -1, g * W + torch.div(at, case["vocab"], rounding_mode="floor")).int())
            res["tokens"].append(torch.where(gone, -1, at % case["vocab"]).int())
        return {name: torch.stack(v) for name, v in res.items()}

    page, KV, n, half = case["page"], case["kv_heads"], case["n"], ROT // 2
    rep, T = case["heads"] // KV, case["n"] * case["seqs"]

    def normed(x, w, pos):
        x = x.double()
        y = x / ((x ** 2).sum(-1, keepdim=True) / HEAD_DIM + EPS).sqrt() * (w.double() + 1.0)
        co, si = s["cos"][pos].double(), s["sin"][pos].double()
        lo, hi = y[:, :half].clone(), y[:, half:ROT].clone()
        y[:, :half] = lo * co[:, :half] - hi * si[:, :half]
        y[:, half:ROT] = hi * co[:, half:] + lo * si[:, half:]
        return y

    # every scale that a word can hold, in ascending order
    scales = torch.tensor([(b if b < 64 else (64 + b % 64) * 2.0 ** (b // 64 - 1)) * 2.0 ** -20 for b in range(31 * 64)],
                          dtype=torch.float64, device=DEV)

    def held(y):
        """Values y [n, 256] (64 bits) as the cache holds them."""
        y = y.reshape(-1, 8, 32).float().double().clamp(-2.0 ** 15, 2.0 ** 15)
        least = torch.minimum(y.min(-1).values, torch.zeros((), dtype=torch.float64, device=DEV))
        most = torch.maximum(y.max(-1).values, torch.zeros((), dtype=torch.float64, device=DEV))
        step = scales[torch.searchsorted(scales, (most - least) / 15)][..., None]
        zero = torch.nan_to_num(torch.round(-least[..., None] / step))
        code = torch.nan_to_num(torch.round(y / step) + zero).clamp(0, 15)
        return ((code - zero) * step).reshape(-1, HEAD_DIM)

    def values(rows):
        """Of cached rows [n, 144]."""
        b = rows.long()
        word = b[:, 128::2] + 256 * b[:, 129::2]
        s_, z = scales[torch.div(word, 16, rounding_mode="floor")], (word % 16).double()
        nib = torch.empty((rows.shape[0], HEAD_DIM), dtype=torch.float64, device=DEV)
        nib[:, 0::2], nib[:, 1::2] = (b[:, :128] % 16).double(), torch.div(b[:, :128], 16, rounding_mode="floor").double()
        return ((nib.view(-1, 8, 32) - z[..., None]) * s_[..., None]).reshape(-1, HEAD_DIM)

    out = torch.empty((T, case["heads"] * HEAD_DIM), dtype=torch.float64, device=DEV)
    new = torch.empty((T, 2, KV, HEAD_DIM), dtype=torch.float64, device=DEV)
    for b, ctx in enumerate(_contexts(case)):
        r = slice(b * n, (b + 1) * n)
        pos, old = torch.arange(ctx, ctx + n, device=DEV), torch.arange(ctx, device=DEV)
        ids = s["table"][b].long()[torch.div(old, page, rounding_mode="floor")]
        for g in range(KV):
            part = slice(g * HEAD_DIM, (g + 1) * HEAD_DIM)
            new[r, 0, g], new[r, 1, g] = held(normed(s["k"][r, part], s["kw"], pos)), held(s["v"][r, part])
            K = torch.cat([values(s["data"][0, ids, 0, g, old % page]), new[r, 0, g]])
            V = torch.cat([values(s["data"][0, ids, 1, g, old % page]), new[r, 1, g]])
            for h in range(g * rep, (g + 1) * rep):
                x = s["qg"][r, 2 * h * HEAD_DIM:2 * (h + 1) * HEAD_DIM]
                a = normed(x[:, :HEAD_DIM], s["qw"], pos) @ K.t().contiguous() / math.sqrt(HEAD_DIM)
                a[torch.arange(ctx + n, device=DEV).expand(n, -1) > pos[:, None]] = -math.inf
                out[r, h * HEAD_DIM:(h + 1) * HEAD_DIM] = torch.softmax(a, 1) @ V * torch.sigmoid(x[:, HEAD_DIM:].double())
    return {"out": out, "held": new}

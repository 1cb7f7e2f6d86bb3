"""Operators of serving several continuations of shared contexts, as measurable cases.

Three groups that one such program uses together, over the 2B decoder's shapes (8 query / 2 kv heads
of 256, 6 attention layers, vocabulary 248320):

  attention  `q35.attention_core_paged`: q/k norms, rotary, append of the new tokens' keys and values
             to a paged cache, causal attention of those tokens over it, sigmoid gate
  copy, fork, compact
             `q35.pages_copy`, `q35.pages_fork`, `q35.pages_compact`: pages copied; sequences forked,
             dropped and given room (a shared last page is copied); pages moved to the pool's front
  logprobs   `q35.token_logprobs`: log probabilities and ranks of given tokens, the entropy of the
             distribution and its top alternatives

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
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _q35():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-3.5_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q35
    return q35


# ---------------------------------------------------------------- cases

def _att(name, dtype, page, prompts=0, chunk=0, behind=0, drafts=0, draft=0, tokens=0, ctx=1, shared=0, heads=8,
         kv_heads=2, mix=0):
    c = dict(op="attention", dtype=dtype, page=page, prompts=prompts, chunk=chunk, behind=behind, drafts=drafts,
             draft=draft, tokens=tokens, ctx=ctx, shared=shared, heads=heads, kv_heads=kv_heads, mix=mix)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one user's next token, a short conversation in a full-precision cache: latency
        _att("chat_token", "f32", 64, tokens=1, ctx=517),
        # 33 users' next tokens, contexts of mixed lengths up to 131072 tokens, 16-bit cache: the cache's stream
        _att("serve_tokens", "bf16", 32, tokens=33, ctx=131072, mix=3),
        # one long prompt's next chunk behind what is cached already, full-precision cache
        _att("prompt_chunk", "f32", 64, prompts=1, chunk=2048, behind=14336),
        # a mixed serving step over a common system prompt: two prompt chunks, 12 sequences whose 5
        # drafted tokens are checked, 30 that decode one token
        _att("mixed_step", "f16", 16, prompts=2, chunk=500, behind=1500, drafts=12, draft=5, tokens=30, ctx=8192,
             shared=256, mix=5),
        # a few pages brought back beside a running batch
        dict(name="copy_few", op="copy", dtype="f32", layers=6, pages=50, n=3, page=16, kv_heads=2),
        # a preempted group of long sequences: hundreds of pages of every attention layer
        dict(name="copy_many", op="copy", dtype="bf16", layers=6, pages=1300, n=600, page=64, kv_heads=2),
        # a beam search step: 8 beams, some dropped, some doubled
        dict(name="fork_beams", op="fork", dtype="f32", layers=6, pages=120, seqs=8, out=8, tokens=390, grow=1, page=64,
             kv_heads=2, mix=1),
        # many samples from few prompts, with room for the first hundred tokens of each
        dict(name="fork_samples", op="fork", dtype="bf16", layers=6, pages=1200, seqs=3, out=200, tokens=2021, grow=100,
             page=64, kv_heads=2, mix=2),
        # a small pool tidied between requests
        dict(name="compact_small", op="compact", dtype="f32", layers=6, pages=64, seqs=5, tokens=150, page=16, kv_heads=2,
             mix=1),
        # a large pool after most of its sequences ended: pages move to the front, the rest can be returned
        dict(name="compact_large", op="compact", dtype="bf16", layers=2, pages=4000, seqs=70, tokens=2900, page=64,
             kv_heads=2, mix=2),
        # the next token's alternatives for one user
        dict(name="next_token", op="logprobs", dtype="f32", rows=1, vocab=VOCAB, top=20, masked=0, targets=True),
        # the tokens of many samples scored, part of the vocabulary masked off
        dict(name="score_rows", op="logprobs", dtype="f32", rows=700, vocab=VOCAB, top=5, masked=271, targets=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "attention", "copy", "fork", "compact", "logprobs", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "attention":
        heads, kv = rng.choice([(8, 2), (8, 2), (8, 2), (4, 1), (6, 2), (4, 4), (8, 1), (16, 2)])
        kind = rng.choice(["tokens", "drafts", "chunk", "mixed"])
        c = dict(heads=heads, kv_heads=kv, mix=rng.randint(0, 10 ** 6), shared=page * rng.randint(0, 5))
        if kind in ("tokens", "mixed"):
            c.update(tokens=_log(rng, 1, 70), ctx=_log(rng, 1, 20000))
        if kind in ("drafts", "mixed"):
            c.update(drafts=_log(rng, 1, 20), draft=rng.randint(2, 9), ctx=_log(rng, 1, 20000))
        if kind in ("chunk", "mixed"):
            c.update(prompts=rng.randint(1, 3), chunk=_log(rng, 10, 700), behind=rng.choice([0, _log(rng, 1, 6000)]))
        return _att(None, dtype, page, **c)
    layers, kv = rng.choice([1, 2, 6]), rng.choice([1, 2, 4])
    if op == "copy":
        n = _log(rng, 1, 250)
        return dict(op=op, dtype=dtype, layers=layers, pages=2 * n + rng.randint(0, 50), n=n, page=page, kv_heads=kv)
    if op == "fork":
        seqs, out, tokens, grow = _log(rng, 1, 12), _log(rng, 1, 60), _log(rng, 1, 900), rng.choice([0, 1, rng.randint(2, 99)])
        per = tokens // page + 2
        pages = seqs * per + out * (grow // page + 2) + rng.randint(0, 40)
        return dict(op=op, dtype=dtype, layers=layers, pages=pages, seqs=seqs, out=out, tokens=tokens, grow=grow, page=page,
                    kv_heads=kv, mix=rng.randint(0, 10 ** 6))
    if op == "compact":
        seqs, tokens = _log(rng, 1, 30), _log(rng, 1, 900)
        pages = int(seqs * (tokens // page + 1) * rng.uniform(1.0, 2.5)) + 1
        return dict(op=op, dtype=dtype, layers=layers, pages=pages, seqs=seqs, tokens=tokens, page=page, kv_heads=kv,
                    mix=rng.randint(0, 10 ** 6))
    vocab = rng.choice([VOCAB, _log(rng, 30, 200000)])
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, 300), vocab=vocab, top=rng.choice([0, 1, 5, 20, rng.randint(2, 30)]),
                masked=rng.choice([0, min(vocab - 30, rng.randint(0, 999))]), targets=rng.random() < 0.8)


def _lengths(case):
    """(new tokens, cached tokens) of every sequence of an attention case, in an order as requests come."""
    r = random.Random(case["mix"])
    sh = case["shared"]
    seqs = []
    for i in range(case["prompts"]):
        n = case["chunk"] if i == 0 else r.randint(1, case["chunk"])
        seqs.append((n, max(sh, case["behind"] if i == 0 else r.randint(0, case["behind"]))))
    for kind, n in (("drafts", case["draft"]), ("tokens", 1)):
        for i in range(case[kind]):
            seqs.append((n, max(sh, case["ctx"] if i == 0 else _log(r, 1, case["ctx"]))))
    if len(seqs) > 8:
        seqs.append((0, sh))  # a slot that has nothing to do in this step
    r.shuffle(seqs)
    return seqs


def _seq_lens(case):
    r = random.Random(case["mix"])
    return [case["tokens"] if i == 0 else r.randint(1, case["tokens"]) for i in range(case["seqs"])]


def _parents(case):
    r = random.Random(case["mix"] + 1)
    p = [r.randrange(case["seqs"]) for _ in range(case["out"])]
    if len(p) > 5:
        p[r.randrange(len(p))] = -1  # a slot that ends here
    return p


# ---------------------------------------------------------------- inputs

def _pool(g, case, pages, layers=1):
    """The pool's values [layers][pages][2][kv heads][page][256]: keys and values of unit size."""
    shape = (layers, pages, 2, case["kv_heads"], case["page"], HEAD_DIM)
    data = torch.empty(shape, dtype=DTYPES[case["dtype"]], device=DEV)
    for l in range(layers):
        for p0 in range(0, pages, 512):
            part = data[l, p0:p0 + 512]
            part.copy_(torch.randn(part.shape, generator=g, device=DEV))
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
        seqs, page, sh = _lengths(case), case["page"], case["shared"] // case["page"]
        need = [-(-(n + c) // page) - sh for n, c in seqs]
        pages = sh + sum(need) + 3
        ids = torch.randperm(pages, generator=cpu).tolist()
        width = sh + max(need) + 1
        table, at = [], sh
        for k in need:
            table.append(ids[:sh] + ids[at:at + k] + [-1] * (width - sh - k))
            at += k
        T, H, KV = sum(n for n, _ in seqs), case["heads"], case["kv_heads"]
        start = [0]
        for n, _ in seqs:
            start.append(start[-1] + n)
        longest = max(n + c for n, c in seqs)
        ang = torch.arange(longest, dtype=torch.float64)[:, None] * (
            THETA ** (-torch.arange(0, ROT, 2, dtype=torch.float64) / ROT))[None, :]
        ang = torch.cat([ang, ang], 1)
        s.update(data=_pool(g, case, pages), table=_i32(table), start=_i32(start), pos=_i32([c for _, c in seqs]),
                 qg=normal(T, H * 2 * HEAD_DIM), k=normal(T, KV * HEAD_DIM, sigma=0.7), v=normal(T, KV * HEAD_DIM),
                 qw=normal(HEAD_DIM, sigma=0.2, mean=0.6), kw=normal(HEAD_DIM, sigma=0.2),
                 cos=ang.cos().float().to(DEV), sin=ang.sin().float().to(DEV), seqs=seqs)
    elif case["op"] == "copy":
        ids = torch.randperm(case["pages"], generator=cpu)
        s.update(data=_pool(g, case, case["pages"], case["layers"]), src=ids[:case["n"]].int().to(DEV),
                 dst=ids[case["n"]:2 * case["n"]].int().to(DEV))
    elif case["op"] in ("fork", "compact"):
        lens, page = _seq_lens(case), case["page"]
        need = [-(-n // page) for n in lens]
        ids = torch.randperm(case["pages"], generator=cpu).tolist()
        width = max(need) + 1 + -(-case.get("grow", 0) // page)
        table, at = [], 0
        for k in need:
            table.append(ids[at:at + k] + [-1] * (width - k))
            at += k
        s.update(data=_pool(g, case, case["pages"], case["layers"]), table=_i32(table), lens=_i32(lens))
        if case["op"] == "fork":
            s.update(parents=_i32(_parents(case)), grow=_i32([case["grow"]] * case["out"]))
    else:
        R, V = case["rows"], case["vocab"]
        x = torch.empty((R, V), dtype=DTYPES[case["dtype"]], device=DEV)
        for r0 in range(0, R, 64):
            x[r0:r0 + 64] = normal(min(64, R - r0), V, sigma=2.5)
        if case["masked"]:
            x[:, torch.randperm(V, generator=cpu)[:case["masked"]].to(DEV)] = -math.inf
        t = torch.randint(0, V, (R,), generator=cpu).int()
        if R > 3:
            t[R // 2] = -1  # a row without a token to score (padding)
        s.update(x=x, targets=t.to(DEV) if case["targets"] else None)
    if own:
        q = _q35()
        if "data" in s:
            s["pool"] = q.PagePool(s["data"])
        if case["op"] == "attention":
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
            return {"out": out, "pool": s["data"]}
        if op == "copy":
            q.pages_copy(s["pool"], s["src"], s["dst"])
            return {"pool": s["data"]}
        if op == "fork":
            f = q.pages_fork(s["pool"], s["table"], s["lens"], s["parents"], s["grow"])
            return {"table": f.table, "lens": f.lens, "refs": f.refs, "pool": s["data"]}
        if op == "compact":
            c = q.pages_compact(s["pool"], s["table"])
            return {"table": c.table, "refs": c.refs, "used": c.used, "pool": s["data"]}
        r = q.token_logprobs(s["x"], s["targets"], top=s["case"]["top"])
        return {"logprob": r.logprob, "rank": r.rank, "entropy": r.entropy, "top_ids": r.top_ids,
                "top_logprobs": r.top_logprobs}
    return {"attention": _plain_attention, "copy": _plain_copy, "fork": _plain_fork, "compact": _plain_compact,
            "logprobs": _plain_logprobs}[op](s)


def _plain_rotate(x, cos, sin):
    a = x[..., :ROT]
    turned = torch.cat([-a[..., ROT // 2:], a[..., :ROT // 2]], -1)
    return torch.cat([a * cos + turned * sin, x[..., ROT:]], -1)


def _plain_attention(s):
    c, data, page = s["case"], s["data"], s["case"]["page"]
    H, KV = c["heads"], c["kv_heads"]
    rep = H // KV
    out = torch.empty((s["qg"].shape[0], H * HEAD_DIM), device=DEV)
    t0 = 0
    for b, (n, ctx) in enumerate(s["seqs"]):
        if n == 0:
            continue
        rows = slice(t0, t0 + n)
        t0 += n
        at = torch.arange(ctx, ctx + n, device=DEV)
        cos, sin = s["cos"][ctx:ctx + n, None], s["sin"][ctx:ctx + n, None]
        # keys in 64 bits: what the cache's type rounds them to must not hang on the last bit of a sum
        k = s["k"][rows].view(n, KV, HEAD_DIM).double()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * (1.0 + s["kw"].double())
        k = _plain_rotate(k, cos.double(), sin.double()).float()
        pg = s["table"][b][at // page].long()
        data[0, pg, 0, :, at % page] = k.to(data.dtype)
        data[0, pg, 1, :, at % page] = s["v"][rows].view(n, KV, HEAD_DIM).to(data.dtype)
        qg = s["qg"][rows].view(n, H, 2, HEAD_DIM)
        q = qg[:, :, 0]
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * (1.0 + s["qw"])
        q = _plain_rotate(q, cos, sin)
        used = s["table"][b, :-(-(ctx + n) // page)].long()
        kv = data[0, used].float().permute(1, 2, 0, 3, 4).reshape(2, KV, -1, HEAD_DIM)[:, :, :ctx + n]
        q = q.view(n, KV, rep, HEAD_DIM).permute(1, 2, 0, 3).reshape(KV, rep * n, HEAD_DIM)
        p = torch.matmul(q, kv[0].transpose(1, 2)).view(KV, rep, n, ctx + n) * HEAD_DIM ** -0.5
        if n > 1:
            p = p.masked_fill(torch.arange(ctx + n, device=DEV)[None, :] > at[:, None], -math.inf)
        p = (p - p.amax(-1, keepdim=True)).exp_()
        o = torch.matmul(p.view(KV, rep * n, ctx + n), kv[1].contiguous()).view(KV, rep, n, HEAD_DIM)
        o = (o / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).reshape(n, H, HEAD_DIM)
        out[rows] = (o / (1.0 + (-qg[:, :, 1]).exp())).reshape(n, H * HEAD_DIM)
    return {"out": out, "pool": data}


def _plain_copy(s):
    s["data"][:, s["dst"].long()] = s["data"][:, s["src"].long()]
    return {"pool": s["data"]}


def _plain_refs(table, pages):
    refs = torch.zeros(pages + 1, dtype=torch.int32, device=DEV)
    ids = torch.where(table >= 0, table, pages).flatten().long()
    refs.index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    return refs[:pages]


def _plain_fork(s):
    data, table, parents, page = s["data"], s["table"], s["parents"], s["case"]["page"]
    pages, B, width = data.shape[1], parents.numel(), table.shape[1]
    par = parents.clamp(min=0).long()
    lens = torch.where(parents >= 0, s["lens"][par], 0)
    tail = lens % page
    i = torch.arange(B, device=DEV)
    later = ((parents[:, None] == parents[None, :]) & (i[None, :] < i[:, None])).any(1)
    kept = lens // page + ((tail > 0) & ~later)
    col = torch.arange(width, device=DEV)[None, :]
    old = table[par]
    new = torch.where(col < kept[:, None], old, -1)
    refs = _plain_refs(new, pages)
    want = (col >= kept[:, None]) & (col < ((lens + s["grow"] + page - 1) // page)[:, None])
    free = torch.where(refs == 0, torch.arange(pages, device=DEV), 2 * pages).sort().values
    rank = (want.flatten().cumsum(0) - 1).clamp(min=0).view(B, width)
    new = torch.where(want, free[rank].int(), new)
    refs = _plain_refs(new, pages)
    child = ((tail > 0) & later).nonzero().flatten()
    last = (lens // page)[child].long()
    src, dst = old[child, last].long(), new[child, last].long()
    used = (torch.arange(page, device=DEV)[None, :] < tail[child][:, None])[None, :, None, None, :, None]
    data[:, dst] = torch.where(used, data[:, src], data[:, dst])
    return {"table": new, "lens": lens.int(), "refs": refs, "pool": data}


def _plain_compact(s):
    data, table = s["data"], s["table"]
    pages = data.shape[1]
    live = _plain_refs(table, pages) > 0
    used = live.sum()
    i = torch.arange(pages, device=DEV)
    holes = (~live & (i < used)).nonzero().flatten()
    moved = (live & (i >= used)).nonzero().flatten()
    to = i.clone()
    to[moved] = holes
    data[:, holes] = data[:, moved]
    new = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), -1)
    return {"table": new, "refs": _plain_refs(new, pages), "used": used.int().view(1), "pool": data}


def _plain_logprobs(s):
    x, top, t = s["x"].float(), s["case"]["top"], s["targets"]
    R, V = x.shape
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    z = e.sum(1, keepdim=True)
    lse = z.log()
    # -sum p log p with log p = d - lse; p = 0 contributes nothing
    entropy = lse[:, 0] - (torch.where(e > 0, d * e, 0.0).sum(1) / z[:, 0])
    res = {"logprob": None, "rank": None, "entropy": entropy, "top_ids": None, "top_logprobs": None}
    if t is not None:
        at = t.clamp(min=0).long()[:, None]
        lp, xt = (d.gather(1, at) - lse)[:, 0], x.gather(1, at)
        i = torch.arange(V, device=DEV)[None, :]
        rank = ((x > xt) | ((x == xt) & (i < at))).sum(1)
        res["logprob"] = torch.where(t >= 0, lp, 0.0)
        res["rank"] = torch.where(t >= 0, rank, -1).int()
    if top:
        # one whole number per value, larger for a larger logit and, of equal ones, for the lower index
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (V - 1 - torch.arange(V, device=DEV))[None, :]
        ids = V - 1 - (key.topk(top, 1).values & 0xFFFFFFFF)
        res["top_ids"] = ids.int()
        res["top_logprobs"] = d.gather(1, ids) - lse
    return res


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "attention":
        size, H, KV = DTYPES[case["dtype"]].itemsize, case["heads"], case["kv_heads"]
        seqs = [(n, c) for n, c in _lengths(case) if n > 0]
        T = sum(n for n, _ in seqs)
        row = 2 * KV * HEAD_DIM
        read = min(case["shared"], max(c for _, c in seqs)) + sum(c - case["shared"] for _, c in seqs)
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in seqs)
        return {"bytes": read * row * size + T * row * (size + 4) + T * H * 3 * HEAD_DIM * 4 + T * 2 * ROT * 4,
                "flops": 4 * HEAD_DIM * H * pairs}
    if case["op"] in ("copy", "fork", "compact"):
        token = 2 * case["kv_heads"] * HEAD_DIM * DTYPES[case["dtype"]].itemsize * case["layers"]
        if case["op"] == "copy":
            return {"bytes": 2 * case["n"] * case["page"] * token + 8 * case["n"], "flops": 0}
        lens = _seq_lens(case)
        entries = sum(-(-n // case["page"]) for n in lens)
        if case["op"] == "compact":
            # the share of the pages in use that lie behind the new end, if they lie anywhere
            moved = int(entries * (1.0 - entries / case["pages"]))
            return {"bytes": 2 * moved * case["page"] * token + 8 * entries + 4 * case["pages"], "flops": 0}
        par = _parents(case)
        copied = sum(lens[p] % case["page"] for i, p in enumerate(par) if p >= 0 and p in par[:i])
        room = sum(-(-(lens[p] if p >= 0 else 0) // case["page"]) + -(-case["grow"] // case["page"]) for p in par)
        return {"bytes": 2 * copied * token + 4 * (entries + room) + 4 * case["pages"], "flops": 0}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["rows"] * (16 + 8 * case["top"]), "flops": 5 * n}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, s)
    # pages hold what was put there and tables whole numbers: by their definitions, entry by entry
    data = s["data"]
    table = s["table"].tolist() if "table" in s else None
    if case["op"] == "copy":
        moves = [(a, b, case["page"]) for a, b in zip(s["src"].tolist(), s["dst"].tolist())]
        res = {}
    elif case["op"] == "fork":
        new, lens, moves, seen, missing = [], [], [], set(), []
        old = s["lens"].tolist()
        for p, grow in zip(s["parents"].tolist(), s["grow"].tolist()):
            n = old[p] if p >= 0 else 0
            full, tail = divmod(n, case["page"])
            row = list(table[p][:full]) if p >= 0 else []
            if tail and p not in seen:
                row.append(table[p][full])
            elif tail:
                missing.append((len(new), full, table[p][full], tail))
            seen.add(p)
            new.append(row)
            lens.append((n, -(-(n + grow) // case["page"])))
        taken = {e for row in new for e in row}
        free = iter(e for e in range(case["pages"]) if e not in taken)
        for row, (_, total) in zip(new, lens):
            row += [next(free) for _ in range(total - len(row))]
        moves = [(a, new[j][at], tail) for j, at, a, tail in missing]
        new = [row + [-1] * (len(table[0]) - len(row)) for row in new]
        res = {"table": _i32(new), "lens": _i32([n for n, _ in lens]), "refs": _exact_refs(new, case["pages"])}
    else:
        live = sorted({e for row in table for e in row if e >= 0})
        n = len(live)
        holes = [e for e in range(n) if e not in set(live)]
        to = dict(zip([e for e in live if e >= n], holes))
        moves = [(a, b, case["page"]) for a, b in to.items()]
        new = [[to.get(e, e) for e in row] for row in table]
        res = {"table": _i32(new), "refs": _exact_refs(new, case["pages"]), "used": _i32([n])}
    after = data.clone()
    for a, b, tokens in moves:
        after[:, b, :, :, :tokens] = data[:, a, :, :, :tokens]
    res["pool"] = after.double()
    return res


def _exact_refs(table, pages):
    count = [0] * pages
    for row in table:
        for e in row:
            if e >= 0:
                count[e] += 1
    return _i32(count)


def _exact_attention(case, s):
    page, KV = case["page"], case["kv_heads"]
    rep = case["heads"] // KV
    pool = s["data"].double()
    kind = s["data"].dtype
    outs = []
    row = 0
    half = ROT // 2

    def normed(x, w, pos):
        x = x.double()
        y = x / ((x ** 2).sum(-1, keepdim=True) / HEAD_DIM + EPS).sqrt() * (w.double() + 1.0)
        c, si = s["cos"][pos].double(), s["sin"][pos].double()
        lo, hi = y[:, :half].clone(), y[:, half:ROT].clone()
        y[:, :half] = lo * c[:, :half] - hi * si[:, :half]
        y[:, half:ROT] = hi * c[:, half:] + lo * si[:, half:]
        return y

    for b, (n, ctx) in enumerate(s["seqs"]):
        if n == 0:
            continue
        pos = torch.arange(ctx, ctx + n, device=DEV)
        ids = s["table"][b].long()[torch.arange(ctx + n, device=DEV) // page]
        slot = torch.arange(ctx + n, device=DEV) % page
        o = []
        for g in range(KV):
            part = slice(g * HEAD_DIM, (g + 1) * HEAD_DIM)
            # the cache holds values of its own type
            pool[0, ids[ctx:], 0, g, slot[ctx:]] = normed(s["k"][row:row + n, part], s["kw"], pos).float().to(kind).double()
            pool[0, ids[ctx:], 1, g, slot[ctx:]] = s["v"][row:row + n, part].to(kind).double()
            K, V = pool[0, ids, 0, g, slot], pool[0, ids, 1, g, slot]
            for h in range(g * rep, (g + 1) * rep):
                x = s["qg"][row:row + n, 2 * h * HEAD_DIM:2 * (h + 1) * HEAD_DIM]
                a = normed(x[:, :HEAD_DIM], s["qw"], pos) @ K.t().contiguous() / math.sqrt(HEAD_DIM)
                a[torch.arange(ctx + n, device=DEV).expand(n, -1) > pos[:, None]] = -math.inf
                o.append(torch.softmax(a, 1) @ V * torch.sigmoid(x[:, HEAD_DIM:].double()))
        outs.append(torch.cat(o, 1))
        row += n
    return {"out": torch.cat(outs), "pool": pool}


def _exact_logprobs(case, s):
    res = {"logprob": None, "rank": None, "entropy": None, "top_ids": None, "top_logprobs": None}
    parts = {k: [] for k in res}
    for r0 in range(0, case["rows"], 64):
        x = s["x"][r0:r0 + 64].double()
        lp = torch.log_softmax(x, 1)
        parts["entropy"].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(1))
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        parts["top_ids"].append(order[:, :case["top"]].int())
        parts["top_logprobs"].append(lp.gather(1, order[:, :case["top"]]))
        if s["targets"] is not None:
            t = s["targets"][r0:r0 + 64]
            hit = order == t[:, None]
            rank = hit.int().argmax(1)
            parts["rank"].append(torch.where(t >= 0, rank, -1).int())
            parts["logprob"].append(torch.where(t >= 0, lp.gather(1, t.clamp(min=0).long()[:, None])[:, 0], 0.0))
    for k, v in parts.items():
        if v and (case["top"] or not k.startswith("top")):
            res[k] = torch.cat(v)
    return res

"""Plain forms in 64 bits of the paged cache's operators and the token scores (numpy and CPU torch)."""
import numpy as np
import torch

HD = 256
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def normed(x, w, cos, sin, rot, eps):
    """RMSNorm (1 + w) and rotary of rows x [n, 256] at positions whose tables are cos / sin [n, rot]."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * (1.0 + w.astype(np.float64))
    h = rot // 2
    lo, hi = y[:, :h].copy(), y[:, h:rot].copy()
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    y[:, :h] = lo * c[:, :h] - hi * s[:, :h]
    y[:, h:rot] = hi * c[:, h:] + lo * s[:, h:]
    return y


def rounded(x, dtype):
    """x (f64) as the cache holds it: to f32, then to the cache's type, both to nearest even."""
    return torch.from_numpy(np.ascontiguousarray(x)).float().to(TORCH[dtype])


def attention(dims, pool, layer, qg, k, v, start, pos, table, qw, kw, cos, sin):
    """pool: CPU tensor, updated in place.  Returns (out f64 [T, heads*256], NaN in rows of no sequence;
    per-row tolerance [T]).

    The tolerance: an f32 dot product of 256 terms is off by about sqrt(256) 2^-24 = 2^-20 of its size (products
    of 22 bits and more add less), so a weight e^s is off by |s| 2^-20; the exponential, the running
    rescales and the sums over keys add a few 2^-22 each.  Weights sum to 1 and an error counts in the
    numerator and the denominator: 2 (max |s| + 2) 2^-20 max |v|, and a margin of 2 for what the 2^-20 is a
    standard deviation of."""
    dt = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[pool.dtype]
    H, KV, page = dims.attn_heads, dims.kv_heads, pool.shape[4]
    rep = H // KV
    T = qg.shape[0]
    out, tol = np.full((T, H * HD), np.nan), np.zeros(T)
    for b in range(len(pos)):
        for i in range(start[b + 1] - start[b]):  # append first
            t, p = start[b] + i, pos[b] + i
            for g in range(KV):
                sl = slice(g * HD, (g + 1) * HD)
                pg = int(table[b][p // page])
                y = normed(k[t:t + 1, sl], kw, cos[p:p + 1], sin[p:p + 1], dims.rot_dim, dims.eps)
                pool[layer, pg, 0, g, p % page] = rounded(y, dt)[0]
                pool[layer, pg, 1, g, p % page] = torch.from_numpy(v[t, sl].copy()).to(TORCH[dt])
    for b in range(len(pos)):
        n, p0 = start[b + 1] - start[b], int(pos[b])
        if n == 0:
            continue
        ctx = p0 + n
        ids = torch.tensor([int(table[b][c]) for c in range((ctx + page - 1) // page)])
        rows = slice(start[b], start[b + 1])
        for g in range(KV):
            K = pool[layer, ids, 0, g].reshape(-1, HD)[:ctx].double().numpy()
            V = pool[layer, ids, 1, g].reshape(-1, HD)[:ctx].double().numpy()
            for h in range(g * rep, (g + 1) * rep):
                q = normed(qg[rows, 2 * h * HD:(2 * h + 1) * HD], qw, cos[p0:ctx], sin[p0:ctx], dims.rot_dim, dims.eps)
                s = q @ K.T / 16.0
                s[np.arange(ctx)[None, :] > (p0 + np.arange(n))[:, None]] = -np.inf
                e = np.exp(s - s.max(1, keepdims=True))
                gate = qg[rows, (2 * h + 1) * HD:(2 * h + 2) * HD].astype(np.float64)
                out[rows, h * HD:(h + 1) * HD] = e / e.sum(1, keepdims=True) @ V / (1.0 + np.exp(-gate))
                size = np.abs(np.where(np.isfinite(s), s, 0.0)).max(1)
                tol[rows] = np.maximum(tol[rows], 4.0 * (size + 2.0) * 2.0 ** -20 * np.abs(V).max())
    return out, tol


def fork(table, lens, parents, grow, n_pages, page):
    """(table_out, lens_out, refs, copies [(src, dst, tokens)], short of pages) by the definition."""
    width = len(table[0])
    rows, out_len, want, copies, seen = [], [], [], [], set()
    for j, p in enumerate(parents):
        n = lens[p] if p >= 0 else 0
        full, tail = divmod(n, page)
        row = list(table[p][:full]) if p >= 0 else []
        if tail and p not in seen:
            row.append(table[p][full])
        elif tail:
            copies.append((j, full, table[p][full], tail))
        seen.add(p)
        rows.append(row)
        out_len.append(n)
        want.append(min(width, -(-(n + (grow[j] if grow is not None else 0)) // page)))
    named = {e for r in rows for e in r}
    free = iter([e for e in range(n_pages) if e not in named])
    short = False
    for r, w in zip(rows, want):
        while len(r) < w:
            e = next(free, -1)
            short |= e < 0
            r.append(e)
    rows = [r + [-1] * (width - len(r)) for r in rows]
    refs = [0] * n_pages
    for r in rows:
        for e in r:
            if e >= 0:
                refs[e] += 1
    return rows, out_len, refs, [(s, rows[j][at], t) for j, at, s, t in copies if rows[j][at] >= 0], short


def compact(table, n_pages):
    """(table_out, refs, used, moves [(src, dst)])"""
    live = sorted({e for r in table for e in r if e >= 0})
    n = len(live)
    holes = [e for e in range(n) if e not in set(live)]
    to = dict(zip([e for e in live if e >= n], holes))
    rows = [[to.get(e, e) for e in r] for r in table]
    refs = [0] * n_pages
    for r in rows:
        for e in r:
            if e >= 0:
                refs[e] += 1
    return rows, refs, n, sorted(to.items())


def scores(x, targets, top):
    """x f64 [M, V] -> (logprob, rank, entropy, top_ids, top_logprobs), tolerance left to the caller."""
    M, V = x.shape
    lp = np.full(M, np.nan)
    rank = np.full(M, -1)
    ent = np.zeros(M)
    ids = np.zeros((M, top), np.int64)
    tlp = np.zeros((M, top))
    for m in range(M):
        r = x[m]
        mx = r.max() if not np.isnan(r).any() else np.nan
        with np.errstate(all="ignore"):
            if mx == -np.inf:
                logp = np.full(V, -np.inf)
                ent[m] = 0.0
            else:
                d = r - mx
                z = np.exp(d).sum()
                logp = d - np.log(z)
                p = np.exp(logp)
                ent[m] = -(np.where(p > 0, p * np.where(p > 0, logp, 0.0), 0.0)).sum() if not np.isnan(z) else np.nan
        key = np.where(np.isnan(r), -np.inf, r)
        order = np.lexsort((np.arange(V), -key, np.isnan(r)))
        ids[m], tlp[m] = order[:top], logp[order[:top]]
        if targets is not None:
            t = targets[m]
            if 0 <= t < V:
                lp[m], rank[m] = logp[t], int(np.where(order == t)[0][0])
            elif t < 0:
                lp[m] = 0.0
    return lp, rank, ent, ids, tlp

"""Plain forms in 64 bits of the 4-bit paged cache (numpy): rows of 256 codes and 8 words of a scale and a zero."""
import numpy as np

import paged_ref as R

HD, ROW = 256, 144


def scale_of(bits):
    """The f16 with these bits, the low 4 left out, as f64."""
    return (np.asarray(bits, np.int64) & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)


SCALES = scale_of(np.arange(0, 0x7C00, 16))  # ascending


def pack(y):
    """f32 values [..., 256] -> uint8 [..., 144]."""
    y = np.asarray(y, np.float32)
    g = y.reshape(-1, 8, 32).astype(np.float64)
    fine = np.isfinite(g).all(-1)
    g = np.clip(np.where(fine[..., None], g, 0.0), -32768.0, 32768.0)
    lo, hi = np.minimum(g.min(-1), 0.0), np.maximum(g.max(-1), 0.0)
    at = np.searchsorted(SCALES, (hi - lo) / 15.0)  # the first that is not below
    s = SCALES[at]
    div = np.where(s > 0, s, 1.0)
    z = np.rint(-lo / div)  # (to even)
    c = np.clip(np.rint(g / div[..., None]) + z[..., None], 0, 15)
    c = np.where((fine & (s > 0))[..., None], c, 0.0).astype(np.uint8).reshape(-1, HD)
    z = np.where(s > 0, z, 0.0)
    word = np.where(fine, at * 16 + z.astype(np.int64), 0x7FF0).astype(np.uint16)
    rows = np.concatenate([c[:, 0::2] | c[:, 1::2] << 4, word.view(np.uint8).reshape(-1, 16)], 1)
    return rows.reshape(y.shape[:-1] + (ROW,))


def unpack(rows):
    """uint8 [..., 144] -> the values, f64."""
    b = np.ascontiguousarray(rows).reshape(-1, ROW)
    word = np.ascontiguousarray(b[:, 128:]).view(np.uint16).astype(np.int64)
    c = np.stack([b[:, :128] & 15, b[:, :128] >> 4], -1).reshape(-1, 8, 32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        v = scale_of(word)[..., None] * (c - (word & 15)[..., None])
    return v.reshape(rows.shape[:-1] + (HD,))


def attention(dims, pool, layer, qg, k, v, start, pos, table, qw, kw, cos, sin):
    """As paged_ref.attention over a pool of rows (numpy uint8 [layers, pages, 2, kv heads, page, 144], updated in place),
    with its tolerances: the values are f16 numbers, multiplied as an f16 cache's are."""
    H, KV, page = dims.attn_heads, dims.kv_heads, pool.shape[4]
    rep, T = H // KV, qg.shape[0]
    out, tol = np.full((T, H * HD), np.nan), np.zeros(T)
    for b in range(len(pos)):
        for i in range(start[b + 1] - start[b]):
            t, p = start[b] + i, pos[b] + i
            for g in range(KV):
                sl, pg = slice(g * HD, (g + 1) * HD), int(table[b][p // page])
                pool[layer, pg, 0, g, p % page] = pack(R.normed(k[t:t + 1, sl], kw, cos[p:p + 1], sin[p:p + 1], dims.rot_dim, dims.eps))[0]
                pool[layer, pg, 1, g, p % page] = pack(v[t, sl])
    for b in range(len(pos)):
        n, p0 = start[b + 1] - start[b], int(pos[b])
        if n == 0:
            continue
        ctx, rows = p0 + n, slice(start[b], start[b + 1])
        ids = [int(table[b][c]) for c in range((ctx + page - 1) // page)]
        for g in range(KV):
            K, V = (unpack(pool[layer, ids, i, g].reshape(-1, ROW)[:ctx]) for i in (0, 1))
            for h in range(g * rep, (g + 1) * rep):
                q = R.normed(qg[rows, 2 * h * HD:(2 * h + 1) * HD], qw, cos[p0:ctx], sin[p0:ctx], dims.rot_dim, dims.eps)
                s = q @ K.T / 16.0
                s[np.arange(ctx)[None, :] > (p0 + np.arange(n))[:, None]] = -np.inf
                e = np.exp(s - s.max(1, keepdims=True))
                gate = qg[rows, (2 * h + 1) * HD:(2 * h + 2) * HD].astype(np.float64)
                out[rows, h * HD:(h + 1) * HD] = e / e.sum(1, keepdims=True) @ V / (1.0 + np.exp(-gate))
                size = np.abs(np.where(np.isfinite(s), s, 0.0)).max(1)
                tol[rows] = np.maximum(tol[rows], 4.0 * (size + 2.0) * 2.0 ** -20 * np.abs(V).max())
    return out, tol

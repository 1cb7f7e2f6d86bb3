"""Plain forms in 64 bits of the beams' selection (numpy)."""
import numpy as np


def candidates(x, scores, ended):
    """x f64 [G W, V], scores [G, W], ended [G W] or None -> f64 [G, W V]: every continuation's score, -inf where there is none."""
    G, W = scores.shape
    V = x.shape[1]
    c = np.full((G * W, V), -np.inf)
    for r in range(G * W):
        s = np.float64(scores.reshape(-1)[r])
        if not np.isfinite(s):
            continue
        if ended is not None and ended[r] >= 0:
            if ended[r] < V:
                c[r, ended[r]] = s
            continue
        row = x[r]
        if np.isnan(row).any() or (row == np.inf).any() or row.max() == -np.inf:
            continue
        m = row.max()
        c[r] = s + (row - (m + np.log(np.exp(row - m).sum())))
    return c.reshape(G, W * V)


def select(x, scores, k, ended=None):
    """(scores [G, k] f64, parents, tokens), and the candidates."""
    G, W = scores.shape
    V = x.shape[1]
    c = candidates(x, scores, ended)
    out = np.full((G, k), -np.inf), np.full((G, k), -1), np.full((G, k), -1)
    for g in range(G):
        order = np.argsort(-c[g], kind="stable")[:k]
        order = order[c[g][order] > -np.inf]
        n = len(order)
        out[0][g, :n], out[1][g, :n], out[2][g, :n] = c[g][order], g * W + order // V, order % V
    return out, c


def tolerance(scores, V):
    """A term e^d of a sum is off by 2^-23 (1 + |d|) at most (the hardware's exponential; d and its product with log2 e are each
    rounded to 24 bits), and the terms' mean |d|, weighted as they are in the sum, is at most ln V: ln sum is off by
    2^-23 (1 + ln V), the rest is f64, and the score is rounded to f32 once."""
    return 2.0 ** -23 * (1 + np.log(max(V, 2))) + 2.0 ** -24 * np.abs(scores)


def check(got, x, scores, k, ended=None):
    """got: (scores, parents, tokens) as numpy arrays.  Places whose neighbours are nearer than the sums' error may hold
    either, as long as they lie in different rows (in one row, and between rows of the same values, the order is exact)."""
    G, W = scores.shape
    V = x.shape[1]
    (ws, wp, wt), c = select(x, scores, k, ended)
    gs, gp, gt = got
    assert gs.shape == gp.shape == gt.shape == (G, k)
    none = wp < 0
    assert ((gp < 0) == none).all() and ((gt < 0) == none).all() and (gs[none] == -np.inf).all()
    err = np.abs(np.where(none, 0, gs.astype(np.float64)) - np.where(none, 0, ws))
    tol = tolerance(np.where(none, 0, ws), V)
    assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:4])
    for g in range(G):
        n = int((~none[g]).sum())
        mine = (gp[g, :n].astype(np.int64) - g * W) * V + gt[g, :n]
        assert len(set(mine.tolist())) == n and (gp[g, :n] // W == g).all()
        if np.array_equal(mine, (wp[g, :n] - g * W) * V + wt[g, :n]):
            continue
        for i in np.flatnonzero(mine != (wp[g, :n] - g * W) * V + wt[g, :n]):
            d = abs(c[g][mine[i]] - ws[g, i])
            assert gp[g, i] != wp[g, i] and 0 < d <= 2 * 2.0 ** -23 * (1 + np.log(V)), (g, i, gp[g, i], gt[g, i], wp[g, i], wt[g, i], d)

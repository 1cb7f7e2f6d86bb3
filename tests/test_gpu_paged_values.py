"""Paged attention of values of every size, with what each row and dim may be off by."""
import numpy as np
import pytest
import torch

import paged_ref as R
import q35

pytestmark = pytest.mark.gpu

HD = 256


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def case(seed, dtype, n, ctx, page=32, heads=4, kv=1, score=1.0):
    """One sequence of n new tokens behind ctx; positions' angles are 0 (keys are what the test puts there)."""
    r = np.random.default_rng(seed)
    f = np.float32
    pages = -(-(n + ctx) // page)
    c = dict(dims=q35.make_dims(attn_heads=heads, kv_heads=kv), page=page, n=n, ctx=ctx, kv=kv,
             pool=torch.from_numpy(r.standard_normal((1, pages, 2, kv, page, HD)).astype(f)).to(R.TORCH[dtype]),
             table=[r.permutation(pages).tolist()], qg=r.standard_normal((n, heads * 2 * HD)).astype(f),
             k=r.standard_normal((n, kv * HD)).astype(f), v=r.standard_normal((n, kv * HD)).astype(f),
             qw=np.full(HD, score - 1.0, f), kw=np.zeros(HD, f), cos=np.ones((n + ctx, 64), f), sin=np.zeros((n + ctx, 64), f))
    return c


def rows_of(c):
    """Pages and slots of the cached tokens."""
    t = np.arange(c["ctx"])
    return torch.tensor(np.asarray(c["table"][0])[t // c["page"]]), torch.tensor(t % c["page"])


def put(c, plane, x):
    """x [ctx, kv, 256] as the cached keys (plane 0) or values (1)."""
    pg, sl = rows_of(c)
    c["pool"][0, pg, plane, :, sl] = torch.from_numpy(np.ascontiguousarray(x)).to(c["pool"].dtype)


def run(c, split=None):
    """The call's outputs [n, heads, 256]; split: the tokens of several calls one after another."""
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    pool = q35.PagePool(c["pool"].clone().cuda())
    outs, at = [], 0
    for m in split or [c["n"]]:
        s = slice(at, at + m)
        outs.append(q35.attention_core_paged(c["dims"], pool, 0, d(c["qg"][s]), d(c["k"][s]), d(c["v"][s]), i32([0, m]), i32([c["ctx"] + at]),
                                             i32(c["table"]), d(c["qw"]), d(c["kw"]), d(c["cos"]), d(c["sin"]), check=True))
        at += m
    return torch.cat(outs).cpu().double().numpy().reshape(c["n"], -1, HD)


def exact(c):
    """(out [n, heads, 256], sum_j p_j |v_j| gated, the same shape; largest |score| per (n, heads, 1)) in 64 bits."""
    dims, n, ctx, kv = c["dims"], c["n"], c["ctx"], c["kv"]
    H = dims.attn_heads
    rep = H // kv
    dt = c["pool"].dtype
    pg, sl = rows_of(c)
    old = c["pool"][0, pg, :, :, sl].double().numpy()  # [ctx, 2, kv, 256]
    out, size, top = (np.zeros((n, H, w)) for w in (HD, HD, 1))
    for g in range(kv):
        s = slice(g * HD, (g + 1) * HD)
        kn = R.normed(c["k"][:, s], c["kw"], c["cos"][ctx:], c["sin"][ctx:], dims.rot_dim, dims.eps)
        K = np.concatenate([old[:, 0, g], torch.from_numpy(kn).float().to(dt).double().numpy()])
        V = np.concatenate([old[:, 1, g], torch.from_numpy(c["v"][:, s].copy()).to(dt).double().numpy()])
        for h in range(g * rep, (g + 1) * rep):
            q = R.normed(c["qg"][:, 2 * h * HD:(2 * h + 1) * HD], c["qw"], c["cos"][ctx:], c["sin"][ctx:], dims.rot_dim, dims.eps)
            x = q @ K.T / 16.0
            x[np.arange(ctx + n)[None, :] > (ctx + np.arange(n))[:, None]] = -np.inf
            e = np.exp(x - x.max(1, keepdims=True))
            p = e / e.sum(1, keepdims=True)
            gate = 1.0 / (1.0 + np.exp(-c["qg"][:, (2 * h + 1) * HD:(2 * h + 2) * HD].astype(np.float64)))
            out[:, h], size[:, h] = p @ V * gate, p @ np.abs(V) * gate
            top[:, h, 0] = np.abs(np.where(np.isfinite(x), x, 0.0)).max(1)
    return out, size, top


def bound(c, size, top):
    """What f32 arithmetic may be off by, of sum_j p_j |v_j|.  A score is a sum of 256 products in f32, off by about
    sqrt(256) 2^-24 = 2^-20 of its size at the most: its weight by |s| 2^-20, in the numerator and the denominator.
    The sums over (n + ctx) keys are made 16 or 32 keys at a time, each time rounded (by less than a step, 2^-23), products
    of parts apart (three at most): (n + ctx) / 16 * 3 * 2^-23 if all go one way; the exponential, rescales and gate a
    few 2^-22.  Then a margin of 2."""
    return 2.0 * (2.0 * (top + 4.0) * 2.0 ** -20 + (c["n"] + c["ctx"]) / 16 * 3 * 2.0 ** -23) * size


@pytest.mark.parametrize("n,split", [(40, None), (40, [1] * 5 + [3, 8, 24])])
@pytest.mark.parametrize("dtype,exponent", [("f32", -120), ("f32", -105), ("f32", -92), ("f32", -80), ("f32", 60), ("f32", 110),
                                            ("bf16", -110), ("bf16", 110)])
def test_values_of_any_exponent(dtype, exponent, n, split):
    """All values times a power of two: the outputs are, too.  (Chunks over f32 caches hold values as f16 halves whose
    power of two ends at 2^-100: steps of 2^-124, half a step off at the most.)"""
    c = case(3, dtype, n, 150)
    c["v"] = (c["v"].astype(np.float64) * 2.0 ** exponent).astype(np.float32)
    pg, sl = rows_of(c)
    put(c, 1, c["pool"][0, pg, 1, :, sl].double().numpy() * 2.0 ** exponent)
    want, size, top = exact(c)
    got = run(c, split)
    err = np.abs(got - want)
    tol = bound(c, size, top) + 2.0 ** -124
    assert (err <= tol).all(), float((err / tol).max())

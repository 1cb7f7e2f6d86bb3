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
    """x [ctx, kv or 1, 256] as the cached keys (plane 0) or values (1)."""
    pg, sl = rows_of(c)
    c["pool"][0, pg, plane, :, sl] = torch.from_numpy(np.ascontiguousarray(x)).to(c["pool"].dtype).expand(-1, c["kv"], -1)


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
    """(out [n, heads, 256], what it may be off by) in 64 bits.

    The bound: a score is a sum of 256 products in f32, off by about sqrt(256) 2^-24 = 2^-20 of their size (|s|, and 4
    for products that cancel): so is its weight, in the numerator and the denominator.  The sums over keys are made 16
    or 32 keys at a time, each time rounded (by less than a step, 2^-23) and products of parts apart (three at most):
    (n + ctx) / 16 * 3 * 2^-23 of sum p |v| if all go one way; the exponential, rescales and gate add a few 2^-22, which
    the 4 covers.  f32 chunks hold values as halves: half a step of 2^-39 of the largest that a tile's tokens see, and a
    weight beside a rising largest value 2^-33 of the largest weight: 32 keys' together, 2^-28 of their values.  Then a
    margin of 2."""
    dims, n, ctx, kv = c["dims"], c["n"], c["ctx"], c["kv"]
    H = dims.attn_heads
    rep = H // kv
    dt = c["pool"].dtype
    pg, sl = rows_of(c)
    old = c["pool"][0, pg, :, :, sl].double().numpy()  # [ctx, 2, kv, 256]
    out, tol = np.zeros((n, H, HD)), np.zeros((n, H, HD))
    for g in range(kv):
        s = slice(g * HD, (g + 1) * HD)
        kn = R.normed(c["k"][:, s], c["kw"], c["cos"][ctx:], c["sin"][ctx:], dims.rot_dim, dims.eps)
        K = np.concatenate([old[:, 0, g], torch.from_numpy(kn).float().to(dt).double().numpy()])
        V = np.concatenate([old[:, 1, g], torch.from_numpy(c["v"][:, s].copy()).to(dt).double().numpy()])
        tok = 128 // rep
        ends = ctx + np.minimum((np.arange(n) // tok + 1) * tok, n)
        seen = np.maximum.accumulate(np.abs(V).max(1))[ends - 1][:, None]
        for h in range(g * rep, (g + 1) * rep):
            q = R.normed(c["qg"][:, 2 * h * HD:(2 * h + 1) * HD], c["qw"], c["cos"][ctx:], c["sin"][ctx:], dims.rot_dim, dims.eps)
            x = q @ K.T / 16.0
            hidden = np.arange(ctx + n)[None, :] > (ctx + np.arange(n))[:, None]
            x[hidden] = -np.inf
            e = np.exp(x - x.max(1, keepdims=True))
            p = e / e.sum(1, keepdims=True)
            gate = 1.0 / (1.0 + np.exp(-c["qg"][:, (2 * h + 1) * HD:(2 * h + 2) * HD].astype(np.float64)))
            out[:, h] = p @ V * gate
            ps = p * (np.where(hidden, 0.0, np.abs(x)) + 4.0)
            size = p @ np.abs(V)
            t = 2.0 ** -20 * (ps @ np.abs(V) + ps.sum(1, keepdims=True) * size) + (n + ctx) / 16 * 3 * 2.0 ** -23 * size
            if dt == torch.float32:
                t += 2.0 ** -39 * seen + 2.0 ** -28 * np.median(np.abs(V))
            tol[:, h] = 2.0 * t * gate
    return out, tol


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
    want, tol = exact(c)
    err = np.abs(run(c, split) - want)
    tol += 2.0 ** -124
    assert (err <= tol).all(), float((err / tol).max())


def small_weights(seed, dtype, n, ctx, heads=4, kv=1):
    """Every token asks alike: one key takes half of the weight, thousands of others share the other half, their values all of
    one sign; what is lost of each adds up.  Returns the case, its keys and values [ctx, 1, 256], the query's direction."""
    c = case(seed, dtype, n, ctx, heads=heads, kv=kv)
    r = np.random.default_rng(seed)
    q = r.standard_normal(HD).astype(np.float32)
    c["qg"].reshape(n, heads, 2, HD)[:, :, 0] = q
    unit = R.normed(q[None], c["qw"], c["cos"][:1], c["sin"][:1], 64, c["dims"].eps)[0]
    unit /= np.sqrt((unit ** 2).sum())
    K = r.uniform(-0.5, 0.5, (ctx, 1, 1)) * unit  # (the key's length is its score)
    K[ctx // 2, 0] = np.log(ctx) * unit
    V = r.uniform(1.0, 2.0, (ctx, 1, HD))
    return c, K, V, unit


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,split", [(40, None), (10, [1] * 10)])
@pytest.mark.parametrize("factor", [1.0, 2e4, 2e5, 2e6])
def test_many_small_weights_beside_a_large_value(dtype, factor, n, split):
    """Keys of no weight whose values are much larger than all others', in the first unit of 32 tokens, in the middle, in the
    last."""
    if dtype == "f16" and factor > 2e4:
        pytest.skip("not an f16 value")
    c, K, V, unit = small_weights(5, dtype, n, 2048)
    for t in (7, 1100, 2040):
        K[t, 0], V[t] = -60.0 * unit, V[t] * factor
    put(c, 0, K)
    put(c, 1, V)
    want, tol = exact(c)
    err = np.abs(run(c, split) - want)
    print(dtype, factor, n, "largest error over its bound", float((err / tol).max()), "mean error, relative", float(((run(c, split) - want) / want).mean()))
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("factor", [2e6, 2e7])
def test_many_small_weights_in_a_long_chunk(dtype, factor):
    """As above where every block goes over a thousand tokens: 16384 of 8 heads, among each 512 a key that takes half of their
    weight, among each 100 a large value."""
    c, K, V, unit = small_weights(8, dtype, 64, 16384, heads=32, kv=8)
    K[::512, 0] = np.log(512.0) * unit
    K[16384 // 2, 0] = 0.0
    for t in range(3, 16384, 100):
        K[t, 0], V[t] = -60.0 * unit, V[t] * factor
    put(c, 0, K)
    put(c, 1, V)
    want, tol = exact(c)
    err = np.abs(run(c) - want)
    print(dtype, factor, "largest error over its bound", float((err / tol).max()), "largest relative", float((err / np.abs(want)).max()))
    assert (err <= tol).all(), float((err / tol).max())


def test_values_that_rise_through_the_context():
    """Every 64 tokens' values twenty times the ones before, weights to match: all of them count alike."""
    n, ctx = 40, 640
    c, K, V, unit = small_weights(6, "f32", n, ctx)
    for t in range(ctx):
        V[t] *= 20.0 ** (t // 64)
        K[t, 0] = (30.0 - np.log(20.0) * (t // 64)) * unit
    put(c, 0, K)
    put(c, 1, V)
    want, tol = exact(c)
    err = np.abs(run(c) - want)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("ctx", [2048 - 16, 2048])
def test_values_of_tokens_that_come_later(ctx):
    """A token's value 1e12 times all others', in the chunk's last tile: rows of tiles before it are what they are without it."""
    n = 100  # tiles of 32 tokens
    c, K, V, unit = small_weights(7, "f32", n, ctx)
    put(c, 0, K)
    put(c, 1, V)
    c["v"] = np.abs(c["v"])
    before = run(c)
    c["v"][97] *= 1e12
    got = run(c)
    assert np.array_equal(got[:96], before[:96])
    want, tol = exact(c)
    err = np.abs(got - want)
    assert (err <= tol).all(), float((err / tol).max())

"""How far the beams' sums are off: rows in which one, two or three tokens hold the mass, where errors do not mean out, rows of
equal logits, which are exact, and the order of beams that lie further apart than the bound.

With u = 2^-24: a term e^d, d <= 0 its distance from its lane's highest logit so far, has errors of u |d| from d itself, 1.23 u |d| from
the product with log2 e (rounded, as the constant is) and 2 u from the exponential (one unit in the last place).  The 16 terms of a lane's chunk
are added in f32, four and four: five roundings.  Whenever a running maximum above the term rises, by e, its sum is scaled
by a factor off by u (2 + e).  The distances add up to the term's distance D from the row's highest logit; a maximum rises above
the term of rank r (0: the highest) at most r times, and at most once per chunk of its wave, lane, wave, part and step of the
join: C + 10 times.  All else is f64.  So ln sum e^x is off by
    u (7 + 2 sum p min(r, C + 10) + 2.23 sum p D)
at most, p a term's share of the sum."""
import numpy as np
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def lse(x):
    m = x.max()
    return m + np.log(np.exp(x - m).sum())


def bound(x):
    """Of one row x (f64)."""
    d = x.max() - np.sort(x)[::-1]
    p = np.exp(-d)
    p /= p.sum()
    cap = -(-len(x) // 4096) + 10  # (C: no part has more chunks of a wave than the row has)
    return U * (7 + 2 * (p * np.minimum(np.arange(len(x)), cap)).sum() + 2.23 * (p * d).sum())


def rows(seed, n, V, tokens, dtype):
    """n rows of V logits: `tokens` of them within 1.5 of each other hold all but 10^-3 (or less) of the mass."""
    g = np.random.default_rng(seed)
    x = g.normal(0, 1.0, (n, V)).astype(np.float32)
    top = np.float32(np.log(V) + 0.5 + 7)
    for r in range(n):
        # anywhere, or all within the 16 values that a lane adds up
        at = g.choice(V, tokens, replace=False) if r % 2 else (g.integers(0, V // 64) * 64 + np.arange(tokens)) % V
        x[r, at] = top + g.uniform(0, 1.5, tokens).astype(np.float32)
    return torch.from_numpy(x).cuda().to(DT[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 2, 3])
@pytest.mark.parametrize("n,V", [(64, 1025), (64, 50257), (600, 9000), (16, 248320)])
def test_few_tokens_hold_the_mass(dtype, tokens, n, V):
    x = rows(n + V + tokens, n, V, tokens, dtype)
    ref = x.double().cpu().numpy()
    top, want, tol = ref.max(1), np.array([lse(r) for r in ref]), np.array([bound(r) for r in ref])
    # scores that leave next to nothing of the highest continuation's: its own rounding then hides nothing
    s = (want - top).astype(np.float32)
    r = q35.beam_select(x, torch.from_numpy(s[:, None]).cuda(), 1)
    got, truth = r.scores[:, 0].double().cpu().numpy(), s.astype(np.float64) + top - want
    err = np.abs(got - truth)
    print(dtype, tokens, n, V, "largest error", err.max(), "of", tol.min(), flush=True)
    assert (err <= tol + U * np.abs(truth)).all(), (err.max(), np.argwhere(err > tol)[:4])
    assert (tol < 12 * U).all()  # (what the entry point promises for such rows: 7 10^-7)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 63, 1024, 50257, 248320])
def test_equal_logits_are_exact(dtype, V):
    """Terms of 1 throughout: only f64 is left (a logarithm off by 10^-13)."""
    x = torch.full((3, V), -3.25, device="cuda", dtype=DT[dtype])
    s = np.float32(np.log(V))
    r = q35.beam_select(x, torch.full((3, 1), float(s), device="cuda"), 1)
    assert np.abs(r.scores.double().cpu().numpy() - (np.float64(s) - np.log(V))).max() <= 1e-12 + U * 1e-6


def test_beams_further_apart_than_the_bound_keep_their_order():
    V, G = 20000, 300
    x = rows(5, 2 * G, V, 3, "f32")
    ref = x.double().cpu().numpy()
    top, want, tol = ref.max(1), np.array([lse(r) for r in ref]), np.array([bound(r) for r in ref])
    apart = np.zeros(2 * G)
    apart[1::2] = np.where(np.arange(G) % 2, 1, -1) * 1.1 * (tol[::2] + tol[1::2])
    s = (want - top + apart).astype(np.float32)
    truth = s.astype(np.float64) + top - want
    gap = truth[1::2] - truth[::2]
    clear = np.abs(gap) > tol[::2] + tol[1::2]
    assert clear.sum() > G // 2
    r = q35.beam_select(x, torch.from_numpy(s.reshape(G, 2)).cuda(), 1)
    first = r.parents[:, 0].cpu().numpy() - 2 * np.arange(G)
    assert (first[clear] == (gap[clear] > 0)).all()

"""Token scores on the GPU against their definition in 64 bits (tests/paged_ref.py)."""
import numpy as np
import pytest
import torch

import paged_ref as R
import q35

pytestmark = pytest.mark.gpu
DT = R.TORCH


def check(x, targets, top, **kw):
    """x: CUDA tensor [M, V].  Tolerances: x - max is rounded to f32 (|x - max| 2^-24), the logarithm's
    argument is a sum of f32 exponentials, each off by |d| 2^-23 of itself (the product with log2 e is
    rounded): weighted by e^d, a few 2^-22 in all; the result's own rounding is half a step.  The entropy
    weights d, up to its own size, with those errors."""
    h = x.double().cpu().numpy()
    t = targets.cpu().numpy() if targets is not None else None
    r = q35.token_logprobs(x, targets, top=top, **kw)
    lp, rank, ent, ids, tlp = R.scores(h, t, top)

    def close(got, want, scale):
        got = got.cpu().numpy().astype(np.float64)
        tol = 2.0 ** -21 + 2.0 ** -23 * np.abs(np.where(np.isfinite(want), want, 0.0)) + scale
        with np.errstate(invalid="ignore"):
            ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
        assert ok.all(), (got[~ok][:5], want[~ok][:5])

    close(r.entropy, ent, 2.0 ** -21 * (1 + np.abs(np.nan_to_num(ent))))
    if targets is not None:
        assert r.rank.cpu().tolist() == rank.tolist()
        close(r.logprob, lp, 0.0)
    else:
        assert r.logprob is None and r.rank is None
    if top:
        assert r.top_ids.cpu().tolist() == ids.tolist()
        close(r.top_logprobs, tlp, 0.0)
    else:
        assert r.top_ids is None and r.top_logprobs is None
    return r


def logits(seed, M, V, dtype="f32", sigma=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn((M, V), generator=g, device="cuda") * sigma).to(DT[dtype])


def targets_of(seed, M, V):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, V, M).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,V,top", [(1, 1, 1), (1, 2, 2), (3, 64, 64), (2, 63, 5), (5, 1000, 20), (1, 1025, 64), (1, 4097, 7),
                                     (2, 20000, 1), (7, 50257, 20), (1, 248320, 20), (3, 248321, 0), (1100, 130, 3), (1030, 5000, 33)])
def test_scores(M, V, top, dtype):
    print(M, V, top, dtype, flush=True)
    check(logits(M + V, M, V, dtype), targets_of(V, M, V), top)


def test_without_targets_and_leading_dimensions():
    x = logits(1, 6, 700)
    check(x, None, 4)
    t = targets_of(2, 6, 700)
    a = q35.token_logprobs(x, t, top=4)
    b = q35.token_logprobs(x.view(2, 3, 700), t.view(2, 3), top=4)
    assert b.logprob.shape == (2, 3) and b.top_ids.shape == (2, 3, 4)
    for u, v in zip(a, b):
        assert torch.equal(u.flatten(), v.flatten())
    e = q35.token_logprobs(x[:0], t[:0], top=4)
    assert e.logprob.shape == (0,) and e.top_ids.shape == (0, 4)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,off", [(333, 1), (4099, 3), (9000, 5), (70001, 7)])
def test_strided_and_unaligned_rows(V, off, dtype):
    wide = logits(V, 4, V + 20, dtype)
    wide[:, :off] = float("nan")
    wide[:, off + V:] = float("inf")
    check(wide[:, off:off + V], targets_of(V, 4, V), min(V, 11))


def test_padded_vocabulary_is_not_copied():
    """Rows [B, T, V] cut out of wider ones have one stride: they are read where they are."""
    V, wide = 20001, 20032
    x = logits(9, 6, wide, "bf16").view(2, 3, wide)
    x[..., V:] = float("nan")
    t = targets_of(10, 6, V)
    q35.token_logprobs(x[..., :V], t.view(2, 3), top=5)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    r = q35.token_logprobs(x[..., :V], t.view(2, 3), top=5)
    assert torch.cuda.max_memory_allocated() - before < x.numel() * 2
    want = check(x.view(6, wide)[:, :V], t, 5)  # (a copy's rows begin elsewhere in their 16-byte words: sums in another order)
    for u, v in zip(r, want):
        assert torch.equal(u.flatten(), v.flatten())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties_go_to_the_lowest_id(dtype):
    for V in (100, 3000, 60000):
        x = torch.zeros((3, V), device="cuda", dtype=DT[dtype])
        x[1] = torch.arange(V, device="cuda") % 3
        x[2, V // 2:] = -0.0
        check(x, targets_of(V, 3, V), 64)
        y = (logits(V, 3, V) * 2).round().to(DT[dtype])
        check(y, targets_of(V + 1, 3, V), 50)


def test_ascending_and_descending_rows():
    """Every value displaces the list's last one; and none does after the first."""
    V = 30000
    up = torch.arange(V, device="cuda", dtype=torch.float32) * 0.01
    x = torch.stack([up, up.flip(0)])
    check(x, targets_of(1, 2, V), 64)


def test_one_very_long_row():
    """20 million values: every split of the row is many chunks; the planted largest ones are told, in order."""
    V, n = 20_000_003, 64
    x = -torch.rand((1, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    at = torch.randperm(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))[:n]
    x[0, at] = torch.arange(n, 0, -1, device="cuda", dtype=torch.float32) * 0.25
    t = at[40:41].int()
    r = q35.token_logprobs(x, t, top=n)
    assert torch.equal(r.top_ids[0].long(), at) and int(r.rank) == 40
    lse = torch.logsumexp(x[0].double(), 0)
    p = (x[0].double() - lse).exp()
    ent = -(p * (x[0].double() - lse)).sum()
    # the largest value is 16: differences of up to 17 rounded to f32, and the exponentials' own error, as in check()
    assert abs(float(r.logprob) - float(x[0, at[40]].double() - lse)) <= 2.0 ** -21 + 2.0 ** -23 * 17
    assert abs(float(r.entropy) - float(ent)) <= 2.0 ** -21 * (2 + float(ent)) + 2.0 ** -23 * float(ent)


@pytest.mark.parametrize("V", [1, 2, 5, 63, 70, 1030, 5000])
def test_rows_of_nan_and_infinities(V):
    """NaN, -inf, inf, few numbers in every mixture: the order of ids is still told."""
    g = np.random.default_rng(V)
    x = g.choice(np.array([np.nan, -np.inf, np.inf, -1.5, 2.0, 0.0, -3e38], np.float32), (24, V))
    for m in range(7):
        x[m] = g.choice(np.array([np.nan, -np.inf, np.inf, -1.5, 2.0, 0.0, -3e38], np.float32)[[m, (m + 1) % 7]], V)
    x[7], x[8], x[9] = np.nan, -np.inf, -3.4e38
    t = torch.from_numpy(g.integers(0, V, 24).astype(np.int32)).cuda()
    for top in sorted({1, min(V, 3), min(V, 40), min(V, 64)}):
        check(torch.from_numpy(x).cuda(), t, top)


@pytest.mark.parametrize("top", [1, 2, 20, 33, 63, 64])
def test_largest_values_anywhere(top):
    """The highest alternatives in one part of a long row, in a few, one in each, spread thinner and thinner; among
    them NaN, and rows of few different values."""
    V = 248320
    g = np.random.default_rng(top)
    x = g.standard_normal((8, V)).astype(np.float32)
    x[0, 100000:100064] += 50                    # one part
    x[1, np.arange(64) * 3881] += 50             # everywhere
    x[2, 5000:5040] += 50                        # two parts
    x[2, 240000:240030] += 49
    for i in range(6):                           # 32 here, 16 there, ..
        x[3, 20000 * i:20000 * i + (32 >> i)] += 60 - i
    x[4] = np.sort(x[4])
    x[5] = np.sort(x[5])[::-1]
    x[6] = np.round(x[6])
    x[7, g.permutation(V)[:V // 2]] = np.nan
    for rows in (x, x[:1], x[4:5], x[7:]):
        t = torch.from_numpy(np.full(len(rows), 100003, np.int32)).cuda()
        check(torch.from_numpy(np.ascontiguousarray(rows)).cuda(), t, top)


def test_masked_rows():
    """-inf, the type's lowest value, a single open token, rows with nothing open."""
    inf = float("inf")
    for V in (70, 9001):
        x = logits(V, 7, V)
        x[0, ::2] = -inf
        x[1] = -inf
        x[2] = -inf
        x[2, V - 2] = 3.0
        x[3, 5:] = torch.finfo(torch.float32).min
        x[4] = torch.finfo(torch.float32).min
        x[5, :60] = -inf
        x[6] = 80.0 * x[6]
        t = torch.tensor([1, 3, V - 2, V - 1, 4, 2, 0], dtype=torch.int32, device="cuda")
        check(x, t, 64)
        t[0] = 2  # a masked target
        r = check(x, t, 3)
        assert r.logprob[0] == -inf and r.entropy[1] == 0 and r.logprob[1] == -inf and r.top_ids[1].tolist() == [0, 1, 2]


def test_nan_and_infinity():
    nan, inf = float("nan"), float("inf")
    for V in (90, 9000):
        x = logits(V, 4, V)
        x[0, 17] = nan
        x[1] = nan
        x[2, 40] = inf
        t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
        r = q35.token_logprobs(x, t, top=40)
        assert r.logprob[:3].isnan().all() and r.entropy[:3].isnan().all() and r.top_logprobs[:3].isnan().all()
        assert 17 not in r.top_ids[0].tolist() and r.top_ids[1].tolist() == list(range(40)) and r.top_ids[2, 0] == 40
        assert r.logprob[3].isfinite()
        for tt in ([17, 2, 40, 3], [18, V - 1, 41, 0]):  # targets that are a NaN, lie among NaN, are the infinity
            tt = torch.tensor(tt, dtype=torch.int32, device="cuda")
            want = R.scores(x.double().cpu().numpy(), tt.cpu().numpy(), 1)[1]
            assert q35.token_logprobs(x, tt).rank.tolist() == want.tolist()
        x[0, :V - 5] = nan
        ids = q35.token_logprobs(x, top=10).top_ids[0].tolist()
        assert sorted(ids[:5]) == list(range(V - 5, V)) and ids[5:] == list(range(5))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ranks_at_every_place(dtype):
    """The target is each value of a row with ties in turn: words before, around and behind it; zeros of both signs."""
    V = 97
    x = (logits(8, 1, V, sigma=1.5).round() * torch.where(torch.arange(V, device="cuda") % 2 == 0, 1.0, -1.0)).to(DT[dtype]).repeat(V, 1)
    t = torch.arange(V, dtype=torch.int32, device="cuda")
    r = check(x, t, 5)
    assert sorted(r.rank.tolist()) == list(range(V))
    y = torch.cat([logits(9, V, 4000, dtype), x], 1)
    check(y, t + 4000, 5)


def test_targets_outside():
    x = logits(3, 4, 500)
    t = torch.tensor([-1, 500, 7, -100], dtype=torch.int32, device="cuda")
    r = q35.token_logprobs(x, t)
    assert r.logprob[0] == 0 and r.logprob[3] == 0 and r.logprob[1].isnan() and r.rank.tolist()[:2] == [-1, -1] and r.rank[3] == -1
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        q35.token_logprobs(x, t, check=True)
    t[1] = 499
    q35.token_logprobs(x, t, check=True)


def test_rows_behind_32bit_offsets():
    """9000 bf16 rows of 248320: the last ones lie behind 2^31 values."""
    M, V = 9000, 248320
    x = torch.zeros((M, V), dtype=torch.bfloat16, device="cuda")
    x[-2:] = logits(5, 2, V, "bf16")
    r = q35.token_logprobs(x, torch.full((M,), 9, dtype=torch.int32, device="cuda"), top=2)
    s = check(x[-2:], torch.full((2,), 9, dtype=torch.int32, device="cuda"), 2)
    assert torch.equal(r.top_ids[-2:], s.top_ids) and torch.equal(r.rank[-2:], s.rank)
    assert r.top_ids[:-2].eq(torch.tensor([0, 1], device="cuda")).all() and (r.rank[:-2] == 9).all()
    torch.testing.assert_close(r.logprob[-2:], s.logprob, rtol=2e-6, atol=1e-6)


def test_captured_and_replayed():
    x, t = logits(6, 3, 60001), targets_of(6, 3, 60001)
    q35.token_logprobs(x, t, top=9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = q35.token_logprobs(x, t, top=9)
    for seed in range(3):
        x.copy_(logits(seed + 50, 3, 60001))
        t.copy_(targets_of(seed, 3, 60001))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(r, check(x, t, 9)):
            assert torch.equal(a, b)

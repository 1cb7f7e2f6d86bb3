"""The beams' selection on the GPU against its plain form in 64 bits (tests/beam_ref.py)."""
import numpy as np
import pytest
import torch

import beam_ref as B
import q35

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def run(x, scores, k, ended=None, **kw):
    r = q35.beam_select(x, torch.from_numpy(np.asarray(scores, np.float32)).cuda(), k, ended=i32(ended) if ended is not None else None, **kw)
    return tuple(t.cpu().numpy() for t in r)


def verify(x, scores, k, ended=None, **kw):
    got = run(x, scores, k, ended, **kw)
    B.check(got, x.double().cpu().numpy().reshape(-1, x.shape[-1]), np.asarray(scores, np.float32), k, ended)
    return got


def logits(seed, dtype, rows, V, sigma=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(rows, V, generator=g, device="cuda") * sigma).to(DT[dtype])


def make_scores(seed, G, W):
    return np.random.default_rng(seed).normal(-20, 1.5, (G, W)).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,W,V,k", [
    (1, 1, 1, 1), (1, 1, 5, 3), (1, 4, 248320, 8), (2, 3, 1023, 6), (3, 5, 1025, 10), (1, 8, 50257, 16), (40, 4, 333, 8), (7, 12, 4097, 24), (1, 64, 5000, 64),
    (2, 33, 70001, 33), (5, 1, 32000, 64), (300, 2, 129, 5), (1, 256, 700, 64), (1, 2, 20, 64), (9, 7, 16384, 1), (3, 16, 64, 64),
])
def test_matches_64bit(dtype, G, W, V, k):
    print(dtype, G, W, V, k, flush=True)
    verify(logits(G + W + V + k, dtype, G * W, V), make_scores(k, G, W), k)


def test_three_dimensions_strides_and_alignment():
    x = logits(1, "bf16", 6, 900)
    s = make_scores(1, 2, 3)
    first = run(x, s, 7)
    for y in (x.view(2, 3, 900), torch.cat([x, x], 1)[:, :900], torch.cat([torch.zeros(6, 5, dtype=x.dtype, device="cuda"), x], 1)[:, 5:]):
        for a, b in zip(run(y, s, 7), first):
            np.testing.assert_array_equal(a, b)
    # rows in another order of memory are copied
    for a, b in zip(run(x.t().contiguous().t(), s, 7), first):
        np.testing.assert_array_equal(a, b)
    # scores as a part of a wider tensor
    wide = torch.zeros(2, 9, device="cuda")
    wide[:, 4:7] = torch.from_numpy(s).cuda()
    for a, b in zip(q35.beam_select(x, wide[:, 4:7], 7), first):
        np.testing.assert_array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [2001, 20002, 30000])
def test_same_beams_have_equal_scores(dtype, V):
    """Rows of the same values at other addresses: the order is by beam, then by token, throughout."""
    x = logits(3, dtype, 1, V).expand(5, V).contiguous()
    got = verify(x, np.full((1, 5), -3.0), 12)
    order = np.lexsort((np.arange(V), -x[0].double().cpu().numpy()))
    assert got[1][0].tolist() == [0, 1, 2, 3, 4, 0, 1, 2, 3, 4, 0, 1] or len(set(x[0][order[:3].copy()].tolist())) < 3
    if len(set(x[0][order[:3].copy()].tolist())) == 3:
        assert got[2][0].tolist() == [order[i // 5] for i in range(12)]


def test_equal_logits_go_by_token():
    x = torch.zeros(4, 5000, device="cuda")
    got = verify(x, [[-1.0, -1.0], [-2.0, -1.0]], 20)
    assert got[2].tolist() == [list(range(20))] * 2 and got[1].tolist() == [[0] * 20, [3] * 20]
    x[:, 700:] = 3.0
    x[:, 4000] = -0.0
    got = verify(x, [[-1.0, -1.0], [-2.0, -1.0]], 3)
    assert got[2].tolist() == [[700, 701, 702]] * 2


def test_ended_beams():
    x = logits(5, "f32", 12, 3000)
    s = make_scores(5, 3, 4)
    ended = np.full(12, -1)
    ended[[0, 3, 5, 8, 9, 10, 11]] = [2999, 0, 17, 2, 2, 2, 2]
    got = verify(x, s, 8, ended)
    assert got[0][2, :4].tolist() == sorted(s[2].tolist(), reverse=True) and got[1][2].tolist()[4:] == [-1] * 4
    # ended beams' logits are not read
    x[[0, 3, 5, 8, 9, 10, 11]] = float("nan")
    for a, b in zip(run(x, s, 8, ended), got):
        np.testing.assert_array_equal(a, b)
    # an ended beam that leads stays first, at its own score
    s[0, 0] = -1.0
    got = verify(x, s, 8, ended)
    assert (got[0][0, 0], got[1][0, 0], got[2][0, 0]) == (-1.0, 0, 2999)
    as_rows = run(x, s, 8, ended.reshape(3, 4))
    for a, b in zip(as_rows, got):
        np.testing.assert_array_equal(a, b)


def test_ended_tokens_out_of_range_are_reported():
    x, s = logits(6, "f16", 4, 100), make_scores(6, 1, 4)
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        run(x, s, 4, [-1, 100, -1, 3], check=True)
    got = run(x, s, 4, [-1, 2 ** 31 - 1, -1, 3])
    assert 1 not in got[1]
    run(x, s, 4, [-1, 99, -7, 3], check=True)


def test_dead_beams_and_rows_without_continuations():
    x = logits(7, "bf16", 20, 1500)
    s = make_scores(7, 5, 4)
    s[0] = [0.0, -np.inf, -np.inf, -np.inf]   # a first step
    s[1] = -np.inf                            # an empty group
    s[2] = [np.nan, np.inf, -5.0, -np.inf]
    x[1:4] = float("nan")                     # dead beams' logits are not read
    x[4:8] = float("inf")
    x[8:10] = float("nan")
    x[12] = -float("inf")                     # nothing open
    x[13, 700] = float("nan")
    x[14, 1499] = float("inf")
    x[16:20] = -float("inf")
    x[16, 3] = 2.0                            # few continuations in a group
    x[19, 1400:1402] = -1.0
    got = verify(x, s, 6)
    assert got[1][1].tolist() == [-1] * 6 and got[1][4].tolist().count(-1) == 3
    assert set(got[1][3].tolist()) == {15}


@pytest.mark.parametrize("where", ["front", "back", "spread"])
def test_candidates_in_one_place(where):
    """All of a row's highest values in one part of it, in rising and falling order; one beam holds all that is chosen."""
    x = logits(8, "f32", 8, 100000, sigma=0.1)
    ramp = torch.arange(64, device="cuda").float() * 0.01 + 5
    at = {"front": torch.arange(64), "back": torch.arange(99999, 99935, -1), "spread": torch.arange(64) * 1500 + 7}[where].cuda()
    x[:, at] = ramp
    verify(x, [[-1.0, -1.003, -50.0, -1.0, -1.001, -9.0, -1.0, -40.0]], 64)
    verify(x, [[-1.0] + [-90.0] * 7], 64)


@pytest.mark.parametrize("shift,sigma", [(1e3, 1.0), (-1e4, 30.0), (0.0, 1e-3), (0.0, 300.0)])
def test_logits_of_any_size(shift, sigma):
    x = logits(9, "f32", 6, 9000, sigma) + shift
    verify(x, make_scores(9, 2, 3), 9)


def test_scores_far_apart_and_large():
    x = logits(10, "f32", 8, 4000)
    verify(x, [[-1e6, -1e6 + 1, -1e6 - 2, -1e6], [0.0, -300.0, 5.0, -1e30]], 16)


def test_scores_that_swallow_the_logits():
    """A beam's score so large that all of its continuations are equal: its order is that of the logits still."""
    x = logits(14, "bf16", 3, 5000)
    got = run(x, [[-1e30, -1e30, -2e30]], 40)
    order = np.lexsort((np.arange(5000), -x[0].double().cpu().numpy()))[:40]
    assert got[1].tolist() == [[0] * 40] and got[2][0].tolist() == order.tolist() and (got[0] == np.float32(-1e30)).all()
    got = run(x, [[-1e9, -1e9, 0.0]], 12)
    assert got[1].tolist() == [[2] * 12]


@pytest.mark.parametrize("W,k", [(64, 64), (8, 64), (12, 24)])
def test_more_equal_continuations_than_the_choice_ranks(W, k):
    """Equal logits and scores throughout, or in many rows and parts: by row, then by token."""
    x = torch.zeros(W, 30000, device="cuda")
    got = verify(x, np.full((1, W), -2.0), k)
    assert got[1][0].tolist() == [0] * k and got[2][0].tolist() == list(range(k))
    x[:, ::7] = 1.0
    x[1] = logits(15, "f32", 1, 30000, 0.3)[0]
    verify(x, np.full((1, W), -2.0), k)
    half = torch.zeros(W, 30000, dtype=torch.bfloat16, device="cuda")
    half[:, 29000:] = 0.5
    got = verify(half, np.linspace(-2.0, -1.0, W)[None].astype(np.float32), k)
    assert got[1][0].tolist() == [W - 1] * k and got[2][0].tolist() == list(range(29000, 29000 + k))


def test_same_bits_on_every_run():
    x, s = logits(11, "bf16", 64, 30000), make_scores(11, 8, 8)
    first = run(x, s, 16)
    for _ in range(3):
        for a, b in zip(run(x, s, 16), first):
            np.testing.assert_array_equal(a, b)


def test_on_another_stream_and_captured():
    x, s = logits(12, "f32", 8, 20000), torch.from_numpy(make_scores(12, 2, 4)).cuda()
    ended = i32([-1] * 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q35.beam_select(x, s, 8, ended=ended)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = q35.beam_select(x, s, 8, ended=ended)
    for seed in range(4):
        x.copy_(logits(20 + seed, "f32", 8, 20000))
        s.copy_(torch.from_numpy(make_scores(seed, 2, 4)))
        ended.fill_(-1)
        ended[seed] = 5
        graph.replay()
        torch.cuda.synchronize()
        B.check(tuple(t.cpu().numpy() for t in r), x.double().cpu().numpy(), s.cpu().numpy(), 8, ended.cpu().numpy())
        eager = q35.beam_select(x, s, 8, ended=ended)
        assert all(torch.equal(a, b) for a, b in zip(r, eager))


def test_rows_beyond_32bit_offsets():
    """The last rows of 2.2 10^9 values."""
    V = 248320
    x = torch.zeros(9000, V, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    for r0 in range(0, 9000, 500):
        x[r0:r0 + 500].normal_(generator=g)
    s = torch.full((2250, 4), -float("inf"), device="cuda")
    s[-2:] = torch.from_numpy(make_scores(1, 2, 4)).cuda()
    r = q35.beam_select(x, s, 4)
    got = tuple(t[-2:].cpu().numpy() for t in r)
    got[1][:] -= 8992
    B.check(got, x[-8:].double().cpu().numpy(), s[-2:].cpu().numpy(), 4)
    assert (r.parents[:-2] == -1).all()


def test_refusals():
    x, s = logits(13, "f32", 4, 100), torch.zeros(2, 2, device="cuda")
    for bad in (lambda: q35.beam_select(x.double(), s, 3), lambda: q35.beam_select(x, s.double(), 3), lambda: q35.beam_select(x[:3], s, 3),
                lambda: q35.beam_select(x, s, 3, ended=torch.zeros(4, device="cuda")), lambda: q35.beam_select(x.cpu(), s.cpu(), 3)):
        with pytest.raises(AssertionError):
            bad()
    for k in (0, 65):
        with pytest.raises((q35.Q35Error, RuntimeError)):
            q35.beam_select(x, s, k)


@pytest.mark.parametrize("live", [0, 1, 7, 300])
def test_many_groups_with_few_live_beams(live):
    """600 beams of which some score: the others' logits are NaN and hold no place in the work's division."""
    G, W, V = 150, 4, 9000
    x = logits(11, "f16", G * W, V)
    on = np.random.default_rng(live).permutation(G * W)[:live]
    s = np.full(G * W, -np.inf, np.float32)
    s[on] = make_scores(live, G, W).reshape(-1)[:live]
    x[torch.from_numpy(np.flatnonzero(np.isinf(s))).cuda()] = float("nan")
    got = verify(x, s.reshape(G, W), 5)
    assert set(got[1][got[1] >= 0].tolist()) <= set(on.tolist()) and ((got[1] >= 0).sum(1) == np.where(np.isfinite(s).reshape(G, W).any(1), 5, 0)).all()

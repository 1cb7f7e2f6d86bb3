"""Forks of states that are one row per sequence, in place and into other tensors."""
import numpy as np
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def make(seed, shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if dtype in (torch.uint8, torch.int32, torch.int64, torch.int8):
        return torch.randint(0, 100, shape, generator=g, device="cuda").to(dtype)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def want(t, parents):
    return torch.stack([t[j if p < 0 else p] for j, p in enumerate(parents)] + [t[j] for j in range(len(parents), t.shape[0])])


PARENTS = [
    [0], [-1], [1, 0], [1, 2, 3, 0], [3, 3, 3, 3], [0, 0, 1, 2], [1, 1, 2, 2, -1, 0, 6], list(range(9)), [8, 7, 6, 5, 4, 3, 2, 1, 0], [2, 0],
]


@pytest.mark.parametrize("parents", PARENTS, ids=str)
def test_in_place(parents):
    """Chains, cycles, a parent of many, rows that stay."""
    B = max(len(parents), max(parents) + 1)
    states = [make(1, (B, 4, 128, 128)), make(2, (B, 1536, 3)), make(3, (B, 40), torch.int32), make(4, (B, 7), torch.bfloat16), make(5, (B, 5), torch.uint8)]
    ref = [want(t, parents) for t in states]
    got = q35.states_fork(states, i32(parents), check=True)
    for a, b, t in zip(got, ref, states):
        assert a is t and torch.equal(a, b)


@pytest.mark.parametrize("B,seed", [(5, 0), (33, 1), (64, 2), (257, 3), (1000, 4), (4096, 5)])
def test_many_rows(B, seed):
    r = np.random.default_rng(seed)
    parents = r.integers(-1, B, B)
    states = [make(seed, (B, 257)), make(seed, (B, 64, 33), torch.float16), make(seed, (B, 3, 3), torch.uint8)]
    ref = [want(t, parents) for t in states]
    q35.states_fork(states, i32(parents), check=True)
    for a, b in zip(states, ref):
        assert torch.equal(a, b)


def test_every_size_of_a_row():
    for n in (1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 255, 256, 1000, 4095, 4096, 4097, 40000):
        states = [make(n, (6, n), torch.uint8), make(n, (6, n))]
        parents = [5, 0, 1, -1, 1, 2]
        ref = [want(t, parents) for t in states]
        q35.states_fork(states, i32(parents))
        for a, b in zip(states, ref):
            assert torch.equal(a, b), n


def test_into_other_tensors():
    """More rows or fewer than there were; rows of no parent and rows behind stay as they were."""
    for parents in ([2, 0, 0, -1, 1, 2, 2], [1], [0, 1, 2]):
        states = [make(1, (3, 1000)), make(2, (3, 31), torch.float16)]
        out = [make(3, (9, 1000)), make(4, (9, 31), torch.float16)]
        ref = [torch.stack([s[p] if p >= 0 else o[j] for j, p in enumerate(parents)] + list(o[len(parents):])) for s, o in zip(states, out)]
        before = [s.clone() for s in states]
        got = q35.states_fork(states, i32(parents), out=out, check=True)
        assert all(a is b for a, b in zip(got, out))
        for a, b, s, t in zip(out, ref, states, before):
            assert torch.equal(a, b) and torch.equal(s, t)


def test_slices_of_a_cache():
    """The first tokens of contiguous caches [B][heads][tmax][256], a state for each head; what lies behind stays."""
    B, heads, tmax, n = 6, 2, 50, 37
    cache = make(7, (B, heads, tmax, 256))
    parents = [3, 3, 0, 1, -1, 5]
    ref = cache.clone()
    ref[:, :, :n] = torch.stack([cache[j if p < 0 else p, :, :n] for j, p in enumerate(parents)])
    q35.states_fork([cache[:, h, :n] for h in range(heads)], i32(parents), check=True)
    assert torch.equal(cache, ref)


def test_more_states_than_one_launch_takes():
    states = [make(i, (5, 17 + i)) for i in range(150)]
    parents = [4, 0, 0, 3, 2]
    ref = [want(t, parents) for t in states]
    q35.states_fork(states, i32(parents))
    for a, b in zip(states, ref):
        assert torch.equal(a, b)


def test_parents_out_of_range_stay_and_are_reported():
    t = make(1, (4, 100))
    ref = want(t, [1, -1, -1, 0])
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        q35.states_fork([t], i32([1, 4, -2, 0]), check=True)
    assert torch.equal(t, ref)
    q35.states_fork([t], i32([0, 1, 2, 3]), check=True)


def test_nothing_to_do():
    t = make(1, (4, 100))
    ref = t.clone()
    q35.states_fork([], i32([1, 0]))
    q35.states_fork([t], i32([]))
    q35.states_fork([t, make(2, (4, 0))], i32([0, -1, 2, 3]), check=True)
    assert torch.equal(t, ref)


def test_rows_beyond_32bit_offsets():
    """Rows of 700 MB: offsets past 2^32 bytes."""
    t = torch.empty((8, 700 << 20), dtype=torch.uint8, device="cuda")
    for j in range(8):
        t[j].fill_(j)
        t[j, -5:] = torch.arange(5, device="cuda", dtype=torch.uint8) + 10 * j
    parents = [7, 0, 2, 1, 4, 6, 5, 7]
    q35.states_fork([t], i32(parents), check=True)
    for j, p in enumerate(parents):
        assert (t[j, :-5] == p).all() and t[j, -5:].tolist() == [10 * p + i for i in range(5)]


def test_captured_and_replayed():
    states = [make(1, (8, 4, 128, 128)), make(2, (8, 1536, 3))]
    first = [t.clone() for t in states]
    parents = i32([0] * 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q35.states_fork(states, i32(range(8)))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q35.states_fork(states, parents)
    r = np.random.default_rng(0)
    for _ in range(4):
        for t, f in zip(states, first):
            t.copy_(f)
        p = r.integers(-1, 8, 8)
        parents.copy_(torch.from_numpy(p).int())
        graph.replay()
        torch.cuda.synchronize()
        for t, f in zip(states, first):
            assert torch.equal(t, want(f, p))


def test_refusals():
    t = make(1, (4, 6))
    for bad in (lambda: q35.states_fork([t, make(2, (3, 6))], i32([0])), lambda: q35.states_fork([t], i32([0]), out=[make(2, (4, 5))]),
                lambda: q35.states_fork([t], i32([0]), out=[make(2, (4, 6), torch.float16)]), lambda: q35.states_fork([t], i32([0, 1]), out=[make(2, (1, 6))]),
                lambda: q35.states_fork([t], i32([0, 1, 2, 3, 0])), lambda: q35.states_fork([t], torch.zeros(2, device="cuda")),
                lambda: q35.states_fork([make(1, (6, 4)).t()], i32([0])), lambda: q35.states_fork([t], i32([0]), out=[])):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(q35.Q35Error, match="Q35_E_ARG"):
        q35.states_fork([t, make(2, (4, 5)), t], i32([1, 0]))
    with pytest.raises(q35.Q35Error, match="Q35_E_ARG"):
        q35.states_fork([t[:3]], i32([0, 1]), out=[t[1:]])

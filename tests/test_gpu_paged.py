"""Paged caches on the GPU: attention of new tokens over pages, forks, copies and compaction of pages,
against plain forms in 64 bits (tests/paged_ref.py)."""
import zlib

import numpy as np
import pytest
import torch

import paged_ref as R
import q35

pytestmark = pytest.mark.gpu

L = q35._lib
HD = 256
DT = R.TORCH


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def make_attention(seed, dtype, page, heads, kv, seqs, layers=1, layer=0, extra=3, rot=64, width_extra=1, fill=None, shared=0):
    """seqs: (new, cached) per sequence.  Returns a dict of host arrays and the pool (CPU tensor)."""
    r = np.random.default_rng(seed)
    need = [-(-(n + c) // page) - shared for n, c in seqs]
    n_pages = shared + sum(max(k, 0) for k in need) + extra
    ids = r.permutation(n_pages).tolist()
    width = max(1, shared + max(need)) + width_extra
    table, at = [], shared
    for k in need:
        k = max(k, 0)
        table.append(ids[:shared] + ids[at:at + k] + [-1] * (width - shared - k))
        at += k
    T = sum(n for n, _ in seqs)
    start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int64)
    pos = [c for _, c in seqs]
    cap = max(n + c for n, c in seqs)
    dims = q35.make_dims(attn_heads=heads, kv_heads=kv, rot_dim=rot)
    ang = np.arange(cap)[:, None] * (1e7 ** (-np.arange(0, rot, 2) / rot))[None, :]
    ang = np.concatenate([ang, ang], 1)
    f = np.float32
    pool = torch.from_numpy(r.standard_normal((layers, n_pages, 2, kv, page, HD)).astype(f)).to(DT[dtype])
    if fill is not None:  # what no token of a sequence occupies
        used = torch.zeros((n_pages, page), dtype=torch.bool)
        for b, (n, c) in enumerate(seqs):
            for p in range(n + c):
                used[table[b][p // page], p % page] = True
        pool[:, ~used.any(1)] = fill
        pool = torch.where(used[None, :, None, None, :, None], pool, torch.tensor(fill, dtype=pool.dtype))
    return dict(dims=dims, pool=pool, layer=layer, qg=r.standard_normal((T, heads * 2 * HD)).astype(f),
                k=(0.7 * r.standard_normal((T, kv * HD))).astype(f), v=r.standard_normal((T, kv * HD)).astype(f),
                start=start, pos=pos, table=table, qw=(0.5 + 0.2 * r.standard_normal(HD)).astype(f),
                kw=(0.2 * r.standard_normal(HD)).astype(f), cos=np.cos(ang).astype(f), sin=np.sin(ang).astype(f))


def run_attention(c, **kw):
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    pool = q35.PagePool(c["pool"].clone().cuda())
    args = (c["dims"], pool, c["layer"], d(c["qg"]), d(c["k"]), d(c["v"]), i32(c["start"]), i32(c["pos"]), i32(c["table"]),
            d(c["qw"]), d(c["kw"]), d(c["cos"]), d(c["sin"]))
    return q35.attention_core_paged(*args, **kw), pool


def check_attention(c, out, pool):
    ref_pool = c["pool"].clone()
    want, tol = R.attention(c["dims"], ref_pool, c["layer"], c["qg"], c["k"], c["v"], c["start"], c["pos"], c["table"],
                            c["qw"], c["kw"], c["cos"], c["sin"])
    got = out.cpu().numpy().astype(np.float64)
    err = np.abs(got - want).max(1)
    bad = ~(err <= tol)
    assert not bad.any(), (np.where(bad)[0][:8], err[bad][:8], tol[bad][:8])
    # the appended rows and everything else, bit for bit
    a, b = pool.data.cpu(), ref_pool
    same = (a == b) | (a.isnan() & b.isnan())
    assert same.all(), same.logical_not().nonzero()[:4]
    pool.check()


CASES = [
    # one token of one sequence, from an empty cache on
    ("f32", 64, 8, 2, [(1, 0)]),
    ("bf16", 64, 8, 2, [(1, 1)]),
    ("f16", 16, 8, 2, [(1, 15), (1, 16), (1, 17)]),
    ("f32", 16, 8, 2, [(1, 700), (1, 3), (1, 64), (1, 255)]),
    ("bf16", 256, 8, 2, [(1, 1300), (1, 511), (1, 512), (1, 513)]),
    # drafted tokens and empty sequences
    ("bf16", 32, 8, 2, [(5, 100), (0, 40), (3, 31), (0, 0), (2, 0), (7, 333)]),
    ("f16", 64, 8, 2, [(9, 63), (4, 1)]),
    ("f32", 128, 8, 2, [(2, 900), (8, 126)]),
    # chunks of prompts, from nothing and behind a context; mixed with single tokens
    ("f32", 64, 8, 2, [(70, 0)]),
    ("bf16", 64, 8, 2, [(130, 61)]),
    ("f16", 16, 8, 2, [(33, 7), (1, 200), (64, 0)]),
    ("f32", 16, 8, 2, [(1, 50), (100, 300), (5, 9)]),
    ("bf16", 128, 8, 2, [(257, 129), (1, 1), (16, 16)]),
    # head layouts
    ("bf16", 64, 4, 4, [(1, 200), (17, 5)]),
    ("f32", 64, 8, 1, [(1, 77), (9, 70)]),
    ("f16", 32, 6, 2, [(1, 130), (13, 40)]),
    ("bf16", 16, 16, 1, [(1, 90), (20, 33)]),
    ("f32", 32, 10, 2, [(1, 90), (20, 33)]),
    ("f16", 64, 3, 3, [(1, 90), (40, 0)]),
]


@pytest.mark.parametrize("dtype,page,heads,kv,seqs", CASES)
def test_attention_matches_64bit(dtype, page, heads, kv, seqs):
    print(dtype, page, heads, kv, seqs, flush=True)
    c = make_attention(zlib.crc32(repr((dtype, page, heads, seqs)).encode()) % 1000, dtype, page, heads, kv, seqs)
    out, pool = run_attention(c)
    check_attention(c, out, pool)


LARGER = [
    # chunks whose tiles are cut by several blocks; several tiles; more than 64 and more than 256 sequences
    ("f32", 64, 8, 2, [(300, 900)]),
    ("bf16", 32, 8, 2, [(200, 1500), (90, 0), (1, 2000)]),
    ("f16", 16, 8, 2, [(150, 700), (40, 1200)] + [(1, 37 * i) for i in range(20)]),
    ("f32", 16, 4, 1, [(1, 11 * i % 200) for i in range(70)]),
    ("bf16", 16, 2, 1, [(i % 3, (7 * i) % 90) for i in range(330)]),
    ("f32", 32, 8, 2, [(1, 50)] * 30 + [(28, 400)]),      # up to two tokens a sequence on average, one long
    ("f16", 32, 16, 1, [(1, 300), (2, 30), (3, 170)]),
]


@pytest.mark.parametrize("dtype,page,heads,kv,seqs", LARGER)
def test_attention_larger_batches(dtype, page, heads, kv, seqs):
    print(dtype, page, heads, kv, seqs[:6], len(seqs), flush=True)
    c = make_attention(31, dtype, page, heads, kv, seqs)
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,seqs", [
    (8, 2, [(1, 60)] * 7 + [(8, 300)]),     # two tiles beside single tokens, and a token more
    (8, 2, [(1, 60)] * 7 + [(9, 300)]),
    (8, 2, [(0, 5)] * 20 + [(25, 400)]),    # a long one among empty ones, fewer tokens than sequences
    (16, 1, [(1, 60), (0, 3), (3, 200)]),
    (2, 2, [(32, 40), (33, 90), (1, 7)]),   # one head per kv head: 32 tokens are two tiles
])
def test_attention_few_and_many_tokens_meet(dtype, heads, kv, seqs):
    print(dtype, heads, kv, seqs, flush=True)
    c = make_attention(77, dtype, 32, heads, kv, seqs)
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("dtype,scale", [("f32", 1e-12), ("f32", 1e12), ("f16", 2.0 ** -20), ("f16", 2.0 ** 9), ("bf16", 1e-30), ("bf16", 1e30)])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_values_of_any_size(dtype, scale, n):
    """Values of the cache and the new ones all scaled; f16 reaches its subnormal numbers."""
    c = make_attention(32, dtype, 32, 8, 2, [(n, 200)])
    c["pool"][:, :, 1] = (c["pool"][:, :, 1].double() * scale).to(c["pool"].dtype)
    c["v"] = (c["v"] * np.float32(scale)).astype(np.float32)
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("n", [1, 40])
def test_attention_values_zero_in_places(n):
    """Pages of zeros beside small values (f32: the zeros must not set the values' power of two), uneven rows."""
    c = make_attention(33, "f32", 16, 8, 2, [(n, 150)])
    c["pool"] *= 1e-6
    for p in c["table"][0][1:9:2]:
        c["pool"][:, p] = 0.0
    c["v"][:] *= 1e-6
    check_attention(c, *run_attention(c))
    # every 4 tokens' values two thousand times the 4 before: an error of 2^-37 of the largest is allowed
    c = make_attention(34, "f32", 16, 8, 2, [(n, 60)])
    c["v"][:] *= 1e-3
    for t in range(60):
        c["pool"][:, c["table"][0][t // 16], 1, :, t % 16] *= 2000.0 ** (t // 4 % 3)
    check_attention(c, *run_attention(c))


def test_attention_stream_larger_than_the_last_level_cache():
    """70000 tokens of two f32 heads: the loads that pass the caches by, against the contiguous kernel."""
    ctx, page = 70000, 64
    dims = q35.dims_2b()
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    n = -(-(ctx + 1) // page)
    pool = q35.PagePool(torch.randn((1, n, 2, 2, page, HD), generator=g, device="cuda"))
    table = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().cuda()[None]
    kc, vc = (pool.data[0, table[0].long(), i].permute(1, 0, 2, 3).reshape(1, 2, -1, HD).contiguous() for i in (0, 1))
    qg, k, v, qw, kw = rnd(1, 4096), rnd(1, 512), rnd(1, 512), rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    cos, sin = (torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, kc.shape[2]))
    out = q35.attention_core_paged(dims, pool, 0, qg, k, v, i32([0, 1]), i32([ctx]), table, qw, kw, cos, sin, check=True)
    want = q35.attention_core_decode(dims, qg, k, v, qw, kw, kc, vc, i32([ctx]), cos, sin, check=True)
    # both sum 70001 f32 terms of weight 1 in all, off by a few 2^-20 of the scores' size (tests/paged_ref.py)
    torch.testing.assert_close(out, want, rtol=0, atol=4 * 12 * 2.0 ** -20 * float(vc.abs().max()))
    assert float((out - want).abs().max()) < 1e-5
    p = int(table[0, ctx // page])
    torch.testing.assert_close(pool.data[0, p, 0, :, ctx % page], kc[0, :, ctx], rtol=2e-6, atol=1e-6)
    assert torch.equal(pool.data[0, p, 1, :, ctx % page], v.view(2, HD))


def test_attention_one_sequence_in_a_padded_call():
    """One sequence whose rows are fewer than the call's (a captured chunk's shape), down to none."""
    for n in (0, 1, 9, 60):
        c = make_attention(35, "bf16", 32, 8, 2, [(60, 70)])
        c["start"] = np.array([0, n])
        full = torch.full((60, 2048), 4.0, device="cuda")
        out, pool = run_attention(c, out=full)
        assert (out[n:] == 4.0).all()
        cut = dict(c, qg=c["qg"][:n], k=c["k"][:n], v=c["v"][:n])
        check_attention(cut, out[:n], pool)


def test_attention_starts_that_fall_are_refused():
    c = make_attention(36, "f32", 32, 8, 2, [(5, 40), (40, 20), (3, 9)])
    bad = dict(c, start=np.array([0, 45, 5, 48]))
    out, pool = run_attention(bad, out=torch.full((48, 2048), 6.0, device="cuda"))
    assert (out == 6.0).all()
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        pool.check()
    for start in ([0, 5, 45, 49], [-1, 5, 45, 48], [3, 5, 45, 48]):  # past the rows, before them, rows without a sequence
        out, pool = run_attention(dict(c, start=np.array(start)), out=torch.full((48, 2048), 6.0, device="cuda"))
        if start[0] == 3:
            assert (out[:3] == 6.0).all() and not (out[3:] == 6.0).any()
            pool.check()
        else:
            with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
                pool.check()
            assert (out[45:] == 6.0).all() if start[0] == 0 else (out[:5] == 6.0).all()


def test_attention_same_bits_on_every_run():
    c = make_attention(37, "f16", 16, 8, 2, [(1, 700), (90, 333), (5, 100), (1, 0)])
    first = run_attention(c)[0]
    for _ in range(3):
        assert torch.equal(run_attention(c)[0], first)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf")])
def test_attention_ignores_what_no_token_occupies(dtype, fill):
    """Infinities and NaN behind the sequences' ends and in other pages reach nothing."""
    c = make_attention(5, dtype, 32, 8, 2, [(1, 40), (3, 30), (40, 21), (1, 0)], fill=fill)
    out, pool = run_attention(c)
    check_attention(c, out, pool)


def test_attention_shared_pages_layers_and_odd_rotary():
    c = make_attention(6, "bf16", 16, 8, 2, [(1, 50), (4, 33), (30, 40)], layers=3, layer=2, shared=2, rot=22)
    out, pool = run_attention(c)
    check_attention(c, out, pool)
    c = make_attention(7, "f32", 16, 8, 2, [(1, 50), (4, 33)], layers=2, layer=1, rot=256)
    check_attention(c, *run_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_large_scores_and_uneven_values(dtype):
    """Scores of hundreds (one key takes all the weight), values spread over three orders."""
    c = make_attention(8, dtype, 32, 8, 2, [(1, 300), (20, 100)])
    c["qw"] = c["qw"] * 20
    c["pool"][:, :, 1] *= torch.from_numpy(10.0 ** np.random.default_rng(1).uniform(-1.5, 1.5, (c["pool"].shape[1], 1, 32, 1))).to(
        c["pool"].dtype)
    check_attention(c, *run_attention(c))


def test_attention_rows_behind_the_last_sequence_stay():
    c = make_attention(9, "bf16", 32, 8, 2, [(3, 40), (20, 5)])
    T = c["start"][-1]
    for name in ("qg", "k", "v"):
        c[name] = np.concatenate([c[name], np.full((6, c[name].shape[1]), np.nan, np.float32)])
    out = torch.full((T + 6, 8 * HD), 7.0, device="cuda")
    got, pool = run_attention(c, out=out)
    assert got is out and (out[T:] == 7.0).all()
    for name in ("qg", "k", "v"):
        c[name] = c[name][:T]
    check_attention(c, out[:T], pool)


def test_attention_strided_rows():
    """Queries, keys and values as columns of one projection's output, out as columns of a wider tensor."""
    c = make_attention(10, "f32", 64, 8, 2, [(1, 100), (37, 20)])
    T = c["start"][-1]
    wide = torch.zeros(T, 8 * 512 + 2 * 512 + 8, device="cuda")
    wide[:, :4096], wide[:, 4096:4608], wide[:, 4608:5120] = (torch.from_numpy(c[n]).cuda() for n in ("qg", "k", "v"))
    out = torch.full((T, 2048 + 64), 3.0, device="cuda")
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    pool = q35.PagePool(c["pool"].clone().cuda())
    q35.attention_core_paged(c["dims"], pool, 0, wide[:, :4096], wide[:, 4096:4608], wide[:, 4608:5120], i32(c["start"]), i32(c["pos"]),
                             i32(c["table"]), d(c["qw"]), d(c["kw"]), d(c["cos"]), d(c["sin"]), out=out[:, 32:2080])
    assert (out[:, :32] == 3.0).all() and (out[:, 2080:] == 3.0).all()
    check_attention(c, out[:, 32:2080], pool)


def test_attention_pages_beyond_32bit_offsets():
    """A pool of 5.4 GB whose pages in use lie behind 2^32 bytes."""
    c = make_attention(11, "bf16", 64, 8, 2, [(1, 200), (30, 70)])
    n = c["pool"].shape[1]
    total = 40000
    data = torch.empty((1, total, 2, 2, 64, HD), dtype=torch.bfloat16, device="cuda")
    data[:, total - n:] = c["pool"].cuda()
    big = dict(c, table=[[e + total - n if e >= 0 else -1 for e in row] for row in c["table"]])
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    pool = q35.PagePool(data)
    out = q35.attention_core_paged(c["dims"], pool, 0, d(c["qg"]), d(c["k"]), d(c["v"]), i32(c["start"]), i32(c["pos"]), i32(big["table"]),
                                   d(c["qw"]), d(c["kw"]), d(c["cos"]), d(c["sin"]))
    pool.check()
    small = q35.PagePool(data[:, total - n:].contiguous())
    check_attention(c, out, small)


def test_attention_bad_positions_and_pages_are_reported():
    """A sequence whose positions leave its table is skipped; the others are right."""
    c = make_attention(12, "f32", 32, 8, 2, [(2, 40), (3, 50), (1, 20)])
    ok = run_attention(c)[0].clone()
    bad = dict(c, pos=[40, 10 ** 6, 20])
    out = torch.full(ok.shape, 5.0, device="cuda")
    got, pool = run_attention(bad, out=out)
    assert torch.equal(got[:2], ok[:2]) and torch.equal(got[5:], ok[5:]) and (got[2:5] == 5.0).all()
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        pool.check()
    pool.check()  # cleared
    for value in (-1, 10 ** 6):
        table = [list(r) for r in c["table"]]
        table[1][0] = value
        table[1][1] = value
        got, pool = run_attention(dict(c, table=table))
        assert torch.equal(got[:2], ok[:2]) and torch.equal(got[5:], ok[5:])
        with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
            pool.check()
    got, pool = run_attention(dict(c, pos=[40, -1, 20]))
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        pool.check()


def test_attention_on_another_stream_and_two_at_once():
    cs = [make_attention(13 + i, "bf16", 32, 8, 2, [(1, 300), (20, 70), (4, 12)]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    res = []
    for _ in range(3):
        res = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                res.append(run_attention(c))
        torch.cuda.synchronize()
        for c, (out, pool) in zip(cs, res):
            check_attention(c, out, pool)


def test_attention_captured_and_replayed():
    """A captured step replayed with other lengths, tables and rows gives the eager call's bits; two graphs
    replayed in turn do not disturb each other."""
    B, T = 4, 30
    shapes = [[(1, 100), (20, 30), (5, 7), (4, 0)], [(7, 3), (0, 0), (1, 230), (22, 200)], [(1, 1), (1, 2), (1, 3), (1, 4)]]
    cs = [make_attention(20 + i, "bf16", 16, 8, 2, s, extra=0, width_extra=0) for i, s in enumerate(shapes)]
    n_pages = max(c["pool"].shape[1] for c in cs)
    width = max(len(c["table"][0]) for c in cs)
    cap = max(c["cos"].shape[0] for c in cs)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def buffers():
        return dict(data=torch.zeros((1, n_pages, 2, 2, 16, HD), dtype=torch.bfloat16, device="cuda"), qg=torch.zeros(T, 4096, device="cuda"),
                    k=torch.zeros(T, 512, device="cuda"), v=torch.zeros(T, 512, device="cuda"), start=i32([0] * (B + 1)), pos=i32([0] * B),
                    table=i32([[-1] * width] * B), out=torch.zeros(T, 2048, device="cuda"), qw=torch.zeros(HD, device="cuda"),
                    kw=torch.zeros(HD, device="cuda"), cos=torch.zeros(cap, 64, device="cuda"), sin=torch.zeros(cap, 64, device="cuda"))

    def load(bf, c):
        n = c["start"][-1]
        bf["data"].zero_()
        bf["data"][:, :c["pool"].shape[1]] = c["pool"].cuda()
        for name in ("qg", "k", "v"):
            bf[name].zero_()
            bf[name][:n] = d(c[name])
        bf["start"].copy_(i32(c["start"]))
        bf["pos"].copy_(i32(c["pos"]))
        bf["table"].fill_(-1)
        bf["table"][:, :len(c["table"][0])] = i32(c["table"])
        for name in ("qw", "kw"):
            bf[name].copy_(d(c[name]))
        for name in ("cos", "sin"):
            bf[name][:c[name].shape[0]] = d(c[name])

    def call(bf, pool):
        return q35.attention_core_paged(cs[0]["dims"], pool, 0, bf["qg"], bf["k"], bf["v"], bf["start"], bf["pos"], bf["table"], bf["qw"], bf["kw"],
                                        bf["cos"], bf["sin"], out=bf["out"])

    two = []
    for _ in range(2):
        bf = buffers()
        pool = q35.PagePool(bf["data"])
        load(bf, cs[0])
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call(bf, pool)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(bf, pool)
        two.append((bf, pool, g))
    for turn in range(3):
        for k, (bf, pool, g) in enumerate(two):
            load(bf, cs[(turn + k) % 3])
            bf["out"].fill_(9.0)
        for bf, pool, g in two:
            g.replay()
        torch.cuda.synchronize()
        for k, (bf, pool, g) in enumerate(two):
            c = cs[(turn + k) % 3]
            n = c["start"][-1]
            check_attention(c, bf["out"][:n], q35.PagePool(bf["data"][:, :c["pool"].shape[1]].contiguous()))
            assert (bf["out"][n:] == 9.0).all()
            pool.check()
            got = bf["out"].clone()
            load(bf, c)
            assert torch.equal(call(bf, pool)[:n], got[:n])


# ---------------------------------------------------------------- pages

def filled(layers, n_pages, kv, page, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn((layers, n_pages, 2, kv, page, HD), generator=g, device="cuda").to(DT[dtype])


@pytest.mark.parametrize("dtype,layers,kv,page,n", [("f32", 1, 1, 16, 1), ("bf16", 3, 2, 64, 5), ("f16", 2, 1, 256, 40), ("f32", 6, 4, 16, 300),
                                                    ("bf16", 1, 1, 16, 257), ("bf16", 1, 1, 16, 256)])
def test_pages_copy(dtype, layers, kv, page, n):
    r = np.random.default_rng(n)
    data = filled(layers, 2 * n + 3, kv, page, dtype)
    ids = r.permutation(2 * n + 3)
    src, dst = ids[:n], ids[n:2 * n]
    want = data.clone()
    want[:, dst] = data[:, src]
    pool = q35.PagePool(data.clone())
    q35.pages_copy(pool, i32(src), i32(dst), check=True)
    assert torch.equal(pool.data, want)
    # one source for several pages
    q35.pages_copy(pool, i32([src[0]] * n), i32(dst), check=True)
    want[:, dst] = data[:, src[:1]]
    assert torch.equal(pool.data, want)
    # between two pools of other sizes
    other = q35.PagePool(filled(layers, n + 1, kv, page, dtype, 1))
    want = other.data.clone()
    to = r.permutation(n + 1)[:n]
    want[:, to] = pool.data[:, src]
    q35.pages_copy(pool, i32(src), i32(to), to=other, check=True)
    assert torch.equal(other.data, want)
    q35.pages_copy(pool, i32([]), i32([]), check=True)


@pytest.mark.parametrize("many", [False, True])
def test_pages_copy_refuses_clashes(many):
    """Pairs that clash or leave the pool are not copied, the others are; both ways of checking."""
    n = 700
    data = filled(1, n, 1, 16, "bf16")
    pairs = [(0, 1), (2, 3), (4, 3), (5, 6), (6, 7), (8, 8), (9, n), (-1, 10), (11, 12), (2, 13), (10 ** 6, 14), (15, -5)]
    good = [(0, 1), (11, 12), (2, 13)]
    if many:
        more = [(20 + i, 320 + i) for i in range(290)]
        pairs, good = pairs + more, good + more
    want = data.clone()
    for s, d in good:
        want[:, d] = data[:, s]
    pool = q35.PagePool(data.clone())
    q35.pages_copy(pool, i32([p[0] for p in pairs]), i32([p[1] for p in pairs]))
    assert torch.equal(pool.data, want)
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        pool.check()
    # in two pools a page number may be source and destination
    other = q35.PagePool(torch.zeros_like(data))
    q35.pages_copy(pool, i32([5, 6, 8]), i32([6, 7, 8]), to=other, check=True)
    for s, d in ((5, 6), (6, 7), (8, 8)):
        assert torch.equal(other.data[:, d], pool.data[:, s])


def random_tables(seed, seqs, tokens, page, n_pages, width):
    r = np.random.default_rng(seed)
    lens = [int(r.integers(0, tokens + 1)) for _ in range(seqs)]
    lens[0] = tokens
    ids = r.permutation(n_pages).tolist()
    table, at = [], 0
    for n in lens:
        k = -(-n // page)
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    assert at <= n_pages
    return table, lens


def check_fork(pool, data, table, lens, parents, grow, short=False):
    page = data.shape[4]
    f = q35.pages_fork(pool, i32(table), i32(lens), i32(parents), i32(grow) if grow is not None else None)
    rows, out_len, refs, copies, is_short = R.fork(table, lens, parents, grow, data.shape[1], page)
    assert f.table.cpu().tolist() == rows
    assert f.lens.cpu().tolist() == out_len and f.refs.cpu().tolist() == refs
    want = data.clone()
    for s, d, t in copies:
        want[:, d, :, :, :t] = data[:, s, :, :, :t]
    assert torch.equal(pool.data, want)
    assert is_short == short
    if short:
        with pytest.raises(q35.Q35Error, match="Q35_E_NOMEM"):
            pool.check()
    pool.check()
    return f


@pytest.mark.parametrize("dtype,page,layers,kv,seqs,tokens,parents,grow", [
    ("f32", 16, 1, 1, 1, 1, [0, 0], None),
    ("bf16", 16, 2, 2, 3, 16, [0, 0, 0, 1, 2], [0, 1, 16, 17, 0]),     # a full page: shared by all
    ("f16", 32, 6, 2, 4, 100, [3, 3, 1, -1, 0, 0, 0], [1] * 7),
    ("bf16", 64, 1, 4, 5, 300, [-1, -1], [0, 200]),                     # all dropped
    ("f32", 256, 2, 1, 2, 255, [1, 0, 0, 1], None),
    ("bf16", 16, 1, 1, 9, 77, [i % 9 for i in range(60)], [i % 40 for i in range(60)]),
])
def test_pages_fork(dtype, page, layers, kv, seqs, tokens, parents, grow):
    width = -(-tokens // page) + (max(grow) // page + 2 if grow else 1)
    n_pages = seqs * (-(-tokens // page)) + len(parents) * (2 + (max(grow) // page if grow else 0)) + 2
    table, lens = random_tables(1, seqs, tokens, page, n_pages, width)
    data = filled(layers, n_pages, kv, page, dtype)
    pool = q35.PagePool(data.clone())
    check_fork(pool, data, table, lens, parents, grow)
    # the same call again from the same table: the same result
    check_fork(pool, pool.data.clone(), table, lens, parents, grow)


def test_pages_fork_many_rows_and_a_large_pool():
    """More rows and bitmap words than threads; a pool of 262144 pages (4.3 GB, free pages at its end)."""
    table, lens = random_tables(3, 900, 40, 16, 2000 * 3, 6)
    data = filled(1, 6000, 1, 16, "bf16")
    r = np.random.default_rng(4)
    parents = [int(p) for p in r.integers(-1, 900, 2500)]
    grow = [int(g) for g in r.integers(0, 20, 2500)]
    check_fork(q35.PagePool(data.clone()), data, table, lens, parents, grow)
    big = q35.PagePool(torch.zeros((1, 262144, 2, 1, 16, HD), dtype=torch.bfloat16, device="cuda"))
    n, B = 262144, 4096
    table = np.arange(n - 5).tolist() + [-1] * 5
    t = i32(np.array(table, np.int32).reshape(B, 64))
    lens = np.full(B, 1024)
    lens[-1] = 59 * 16
    f = q35.pages_fork(big, t, i32(lens), i32(np.arange(B)), i32([0] * (B - 1) + [80]), check=True)
    assert f.table[-1, 59:].tolist() == list(range(n - 5, n)) and torch.equal(f.table[:-1], t[:-1])
    assert (f.refs == 1).all()
    c = q35.pages_compact(big, f.table[1:].contiguous(), check=True)
    assert int(c.used) == n - 64 and int(c.refs[:n - 64].min()) == 1 and int(c.refs[n - 64:].max()) == 0
    assert sorted(c.table.flatten().tolist()) == list(range(n - 64))
    ids = torch.randperm(n, device="cuda")[:600].int()
    q35.pages_copy(big, ids[:300], ids[300:], check=True)


def test_pages_fork_without_enough_pages():
    table, lens = random_tables(5, 3, 40, 16, 12, 8)
    data = filled(2, 12, 1, 16, "bf16")
    check_fork(q35.PagePool(data.clone()), data, table, lens, [0, 0, 0, 1], [60, 60, 0, 60], short=True)


def test_pages_fork_reports_bad_indices():
    table, lens = random_tables(6, 3, 40, 16, 20, 4)
    data = filled(1, 20, 1, 16, "bf16")
    for parents, ll, tt, grow in (([0, 3], lens, table, [0, 0]), ([0, -2], lens, table, [0, 0]), ([1, 0], [lens[0], -1, lens[2]], table, [0, 0]),
                                  ([1, 0], [lens[0], 65, lens[2]], table, [0, 0]), ([0, 0], lens, [[99] + table[0][1:]] + table[1:], [0, 0]),
                                  ([0, 1], lens, table, [1000, 0]), ([0, 1], lens, table, [-3, 0])):
        pool = q35.PagePool(data.clone())
        f = q35.pages_fork(pool, i32(tt), i32(ll), i32(parents), i32(grow))
        with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
            pool.check()
        assert int(f.table.max()) < 20 and int(f.table.min()) >= -1
    f = q35.pages_fork(q35.PagePool(data.clone()), i32(table), i32(lens), i32([0, 7, 1]))
    good = q35.pages_fork(q35.PagePool(data.clone()), i32(table), i32(lens), i32([0, -1, 1]))
    assert torch.equal(f.table, good.table) and torch.equal(f.lens, good.lens) and torch.equal(f.refs, good.refs)


@pytest.mark.parametrize("dtype,page,layers,kv,seqs,tokens,n_pages", [
    ("f32", 16, 1, 1, 1, 1, 1), ("bf16", 16, 2, 2, 3, 40, 50), ("f16", 64, 6, 1, 7, 200, 33), ("bf16", 32, 1, 2, 40, 300, 900),
    ("f32", 256, 2, 1, 2, 600, 70)])
def test_pages_compact(dtype, page, layers, kv, seqs, tokens, n_pages):
    width = -(-tokens // page) + 1
    table, _ = random_tables(2, seqs, tokens, page, n_pages, width)
    if seqs > 2:
        table[2][:1] = table[0][:1]  # a shared page
    data = filled(layers, n_pages, kv, page, dtype)
    pool = q35.PagePool(data.clone())
    c = q35.pages_compact(pool, i32(table), check=True)
    rows, refs, used, moves = R.compact(table, n_pages)
    assert c.table.cpu().tolist() == rows and c.refs.cpu().tolist() == refs and int(c.used) == used
    want = data.clone()
    for s, d in moves:
        want[:, d] = data[:, s]
    assert torch.equal(pool.data, want)


@pytest.mark.parametrize("layers,seqs,tokens,n_pages,width", [(3, 40, 300, 900, 450), (1, 30, 400, 17000, 30), (1, 700, 380, 16384, 24)])
def test_pages_compact_larger(layers, seqs, tokens, n_pages, width):
    """Tables of more entries, pools of more pages than one launch takes, and the largest pool that it takes."""
    table, _ = random_tables(8, seqs, tokens, 16, n_pages, width)
    data = filled(layers, n_pages, 1, 16, "bf16")
    pool = q35.PagePool(data.clone())
    c = q35.pages_compact(pool, i32(table), check=True)
    rows, refs, used, moves = R.compact(table, n_pages)
    assert c.table.cpu().tolist() == rows and c.refs.cpu().tolist() == refs and int(c.used) == used
    s, d = (torch.tensor(v, device="cuda") for v in zip(*moves))
    want = data.clone()
    want[:, d] = data[:, s]
    assert torch.equal(pool.data, want)


@pytest.mark.parametrize("rows,width", [(42, 10), (43, 10), (20, 820), (4096, 4), (1, 16384)])
def test_pages_fork_one_launch_or_two(rows, width):
    """24 copies for each partly filled page: 42 rows are one launch, 43 two; and as many entries, rows as one takes."""
    layers, kv = (6, 2) if rows < 100 and width < 16384 else (1, 1)
    table, lens = random_tables(12, 5, 75, 16, 40, width)
    parents = [i % 4 for i in range(rows)]
    n_pages = 40 + 2 * rows + (width if rows == 1 else 0)
    grow = [(width - 6) * 16] if rows == 1 else [i % 20 for i in range(rows)]
    if rows == 4096:
        table, lens = [r[:4] for r in table], [min(n, 40) for n in lens]
        n_pages = 16384
    data = filled(layers, n_pages, kv, 16, "bf16")
    check_fork(q35.PagePool(data.clone()), data, table, lens, parents, grow)


def test_pages_compact_empty_and_bad_entries():
    data = filled(1, 40, 1, 16, "bf16")
    pool = q35.PagePool(data.clone())
    c = q35.pages_compact(pool, i32([[-1, -1], [-1, -1]]), check=True)
    assert int(c.used) == 0 and (c.table == -1).all() and (c.refs == 0).all() and torch.equal(pool.data, data)
    c = q35.pages_compact(pool, i32([[39, 40], [-2, 3]]))
    assert c.table.tolist() == [[0, -1], [-1, 1]] or c.table.tolist() == [[1, -1], [-1, 0]]
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        pool.check()
    c = q35.pages_compact(pool, i32([list(range(40))]), check=True)  # all in use
    assert int(c.used) == 40 and c.table.tolist() == [list(range(40))]


def test_pages_captured_and_replayed():
    table, lens = random_tables(7, 6, 90, 16, 100, 10)
    data = filled(2, 100, 1, 16, "bf16")
    pool = q35.PagePool(data.clone())
    t, ln, par, grow = i32(table), i32(lens), i32([0] * 6), i32([5] * 6)
    q35.pages_fork(pool, t, ln, par, grow)
    q35.pages_compact(pool, t)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f = q35.pages_fork(pool, t, ln, par, grow)
        c = q35.pages_compact(pool, f.table)
    for parents in ([0, 0, 1, 1, 5, 5], [5, 4, 3, 2, 1, 0], [2, 2, 2, 2, 2, -1]):
        pool.data.copy_(data)
        par.copy_(i32(parents))
        g.replay()
        torch.cuda.synchronize()
        rows, out_len, refs, copies, _ = R.fork(table, lens, parents, [5] * 6, 100, 16)
        assert f.table.cpu().tolist() == rows and f.refs.cpu().tolist() == refs and f.lens.cpu().tolist() == out_len
        want = data.clone()
        for s, d, n in copies:
            want[:, d, :, :, :n] = data[:, s, :, :, :n]
        rows2, refs2, used, moves = R.compact(rows, 100)
        after = want.clone()
        for s, d in moves:
            after[:, d] = want[:, s]
        assert c.table.cpu().tolist() == rows2 and c.refs.cpu().tolist() == refs2 and int(c.used) == used
        assert torch.equal(pool.data, after)
        pool.check()


# ---------------------------------------------------------------- together

def test_beam_search_over_forked_pages():
    """A prompt chunk, then beam search steps - fork, attention of the next tokens, scores, the best
    continuations - against the same search with every beam's cache kept whole by attention_core_prefill."""
    dims = q35.dims_2b()
    page, beams, V, steps, T0 = 16, 4, 500, 12, 37
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    emb, wq, wk, wv = rnd(V, 64), rnd(64, 4096, f=0.125), rnd(64, 512, f=0.125), rnd(64, 512, f=0.125)
    head = rnd(2048, V, f=0.2)
    qw, kw = rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    cos, sin = (torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, 128))
    prompt = torch.randint(0, V, (T0,), generator=g, device="cuda")

    def rows(tok):
        e = emb[tok]
        return e @ wq, e @ wk, e @ wv

    def best(scores, hist, logits, n_live):
        r = q35.token_logprobs(logits, top=beams)
        total = scores[:n_live, None] + r.top_logprobs
        flat = total.flatten()
        top = torch.sort(flat, descending=True, stable=True)
        idx = top.indices[:beams]
        parents = (idx // beams).int()
        tok = r.top_ids.flatten()[idx].long()
        return top.values[:beams], parents, tok

    # pages
    pool = q35.PagePool.empty(1, 64, page=page)
    pool.data.fill_(float("nan"))
    f = q35.pages_fork(pool, i32([[-1] * 5]), i32([0]), i32([-1]), i32([T0]))
    out = q35.attention_core_paged(dims, pool, 0, *rows(prompt), i32([0, T0]), f.lens, f.table, qw, kw, cos, sin)
    scores = torch.zeros(1, device="cuda")
    scores, parents, tok = best(scores, None, out[-1:] @ head, 1)
    lens = i32([T0])
    table = f.table
    seqs = [[int(t)] for t in tok]
    start = i32(list(range(beams + 1)))
    for _ in range(steps):
        f = q35.pages_fork(pool, table, lens, parents, i32([1] * beams))
        table, lens = f.table, f.lens
        out = q35.attention_core_paged(dims, pool, 0, *rows(tok), start, lens, table, qw, kw, cos, sin)
        lens = lens + 1
        scores, parents, tok = best(scores, None, out @ head, beams)
        seqs = [seqs[int(p)] + [int(t)] for p, t in zip(parents, tok)]
    pool.check()

    # whole caches
    def forward(ids):
        kc = torch.zeros(2, 128, HD, device="cuda")
        vc = torch.zeros(2, 128, HD, device="cuda")
        a, b, c = rows(torch.tensor(ids, device="cuda"))
        return q35.attention_core_prefill(dims, a, b, c, qw, kw, kc, vc, 0, cos, sin)[-1:]

    sc = torch.zeros(1, device="cuda")
    sc, par, tk = best(sc, None, forward(prompt.tolist()) @ head, 1)
    ref = [[int(t)] for t in tk]
    for _ in range(steps):
        lg = torch.cat([forward(prompt.tolist() + s) @ head for s in ref])
        sc, par, tk = best(sc, None, lg, beams)
        ref = [ref[int(p)] + [int(t)] for p, t in zip(par, tk)]
    assert seqs == ref
    torch.testing.assert_close(scores, sc, rtol=0, atol=1e-4)

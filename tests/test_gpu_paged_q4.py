"""Paged caches in 4 bits on the GPU: what is appended, attention over it, rows read back, forks, copies and compaction,
against plain forms in 64 bits (tests/q4_ref.py)."""
import zlib

import numpy as np
import pytest
import torch

import paged_ref as R
import q35
import q4_ref as Q

pytestmark = pytest.mark.gpu

HD, ROW = 256, 144


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def d(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def make(seed, page, heads, kv, seqs, layers=1, layer=0, extra=3, rot=64, fill=None, shared=0, sigma=1.0):
    """seqs: (new, cached) per sequence; the pool's rows hold values of size sigma, what no token occupies `fill`."""
    r = np.random.default_rng(seed)
    need = [max(-(-(n + c) // page) - shared, 0) for n, c in seqs]
    n_pages = shared + sum(need) + extra
    ids = r.permutation(n_pages).tolist()
    width = max(1, shared + max(need)) + 1
    table, at = [], shared
    for k in need:
        table.append(ids[:shared] + ids[at:at + k] + [-1] * (width - shared - k))
        at += k
    T, cap = sum(n for n, _ in seqs), max(n + c for n, c in seqs)
    start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int64)
    ang = np.arange(cap)[:, None] * (1e7 ** (-np.arange(0, rot, 2) / rot))[None, :]
    ang = np.concatenate([ang, ang], 1)
    f = np.float32
    pool = Q.pack(sigma * r.standard_normal((layers, n_pages, 2, kv, page, HD)))
    if fill is not None:
        used = np.zeros((n_pages, page), bool)
        for b, (n, c) in enumerate(seqs):
            for p in range(n + c):
                used[table[b][p // page], p % page] = True
        pool = np.where(used[None, :, None, None, :, None], pool, np.uint8(fill))
    return dict(dims=q35.make_dims(attn_heads=heads, kv_heads=kv, rot_dim=rot), pool=pool, layer=layer,
                qg=r.standard_normal((T, heads * 2 * HD)).astype(f), k=(0.7 * r.standard_normal((T, kv * HD))).astype(f),
                v=(sigma * r.standard_normal((T, kv * HD))).astype(f), start=start, pos=[c for _, c in seqs], table=table,
                qw=(0.5 + 0.2 * r.standard_normal(HD)).astype(f), kw=(0.2 * r.standard_normal(HD)).astype(f),
                cos=np.cos(ang).astype(f), sin=np.sin(ang).astype(f))


def run(c, pool=None, **kw):
    pool = q35.PagePool(d(c["pool"])) if pool is None else pool
    return q35.attention_core_paged(c["dims"], pool, c["layer"], d(c["qg"]), d(c["k"]), d(c["v"]), i32(c["start"]), i32(c["pos"]),
                                    i32(c["table"]), d(c["qw"]), d(c["kw"]), d(c["cos"]), d(c["sin"]), **kw), pool


def check(c, out, pool):
    ref = c["pool"].copy()
    want, tol = Q.attention(c["dims"], ref, c["layer"], c["qg"], c["k"], c["v"], c["start"], c["pos"], c["table"], c["qw"], c["kw"],
                            c["cos"], c["sin"])
    err = np.abs(out.cpu().numpy().astype(np.float64) - want).max(1)
    bad = ~(err <= tol)
    assert not bad.any(), (np.where(bad)[0][:8], err[bad][:8], tol[bad][:8])
    got = pool.data.cpu().numpy()
    assert (got == ref).all(), np.argwhere(got != ref)[:4]
    pool.check()


CASES = [
    (64, 8, 2, [(1, 0)]),
    (64, 8, 2, [(1, 1)]),
    (16, 8, 2, [(1, 15), (1, 16), (1, 17), (1, 31), (1, 32)]),
    (16, 8, 2, [(1, 700), (1, 3), (1, 64), (1, 255)]),
    (256, 8, 2, [(1, 1300), (1, 511), (1, 512), (1, 513)]),
    (32, 8, 2, [(5, 100), (0, 40), (3, 31), (0, 0), (2, 0), (7, 333)]),
    (64, 8, 2, [(9, 63), (4, 1)]),
    (64, 8, 2, [(70, 0)]),
    (64, 8, 2, [(130, 61)]),
    (16, 8, 2, [(33, 7), (1, 200), (64, 0)]),
    (128, 8, 2, [(257, 129), (1, 1), (16, 16)]),
    (64, 4, 4, [(1, 200), (17, 5)]),
    (32, 6, 2, [(1, 130), (13, 40)]),
    (16, 16, 1, [(1, 90), (20, 33)]),
    (64, 3, 3, [(1, 90), (40, 0)]),
    (64, 8, 2, [(300, 900)]),
    (32, 8, 2, [(200, 1500), (90, 0), (1, 2000)]),
    (16, 8, 2, [(150, 700), (40, 1200)] + [(1, 37 * i) for i in range(20)]),
    (16, 2, 1, [(i % 3, (7 * i) % 90) for i in range(330)]),
    (32, 8, 2, [(1, 50)] * 30 + [(28, 400)]),
]


@pytest.mark.parametrize("page,heads,kv,seqs", CASES)
def test_attention_matches_64bit(page, heads, kv, seqs):
    print(page, heads, kv, seqs[:6], len(seqs), flush=True)
    c = make(zlib.crc32(repr((page, heads, seqs)).encode()) % 1000, page, heads, kv, seqs)
    check(c, *run(c))


def edge_rows():
    """Rows of values whose codes, scales and zeros lie on borders."""
    r = np.random.default_rng(5)
    g = []
    g.append(np.zeros(32))
    g.append(np.full(32, 3.0))
    g.append(np.full(32, -3.0))
    g.append(np.linspace(-1, 1, 32))
    g.append(np.arange(32) / 2.0 - 3.5)            # ties: the scale is 1.03125 or, cut below, exactly 1
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) - 7.5)
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) - 7.0)
    g.append(np.minimum(np.arange(32) / 2.0, 15.0))
    g.append(np.maximum(-np.arange(32) / 2.0, -15.0))
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) * 2.0 ** -20)   # the smallest scale, and below it
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) * 2.0 ** -24)
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) * 1e-30)
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) * 63 * 2.0 ** -20)  # scales of 6, 7 and 8 bits
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) * 127 * 2.0 ** -10)
    g.append(np.minimum(np.arange(32) / 2.0, 15.0) * 129 * 2.0 ** -10)
    g.append(np.linspace(-32768, 32768, 32))
    g.append(np.linspace(-1e6, 3e38, 32))           # cut
    g.append(np.concatenate([np.full(31, 1e-3), [40000.0]]))
    for bad in (np.nan, np.inf, -np.inf):
        x = r.standard_normal(32)
        x[7] = bad
        g.append(x)
    g += [r.standard_normal(32) * 10.0 ** e for e in np.linspace(-8, 5, 27)]
    rows = np.array(g, np.float32).reshape(-1)
    return np.concatenate([rows, r.standard_normal(-len(rows) % HD).astype(np.float32)]).reshape(-1, HD)


def test_appended_rows_are_the_definition():
    v = edge_rows()
    r = np.random.default_rng(6)
    v = np.concatenate([v, r.standard_normal((150, HD)).astype(np.float32) * np.exp(2 * r.standard_normal((150, 1))).astype(np.float32)])
    T = len(v)
    c = make(1, 16, 1, 1, [(T, 5)], fill=0xAB)
    c["v"] = v
    out, pool = run(c)
    want = c["pool"].copy()
    page = 16
    for t in range(T):
        p = 5 + t
        pg = c["table"][0][p // page]
        want[0, pg, 0, 0, p % page] = Q.pack(R.normed(c["k"][t:t + 1], c["kw"], c["cos"][p:p + 1], c["sin"][p:p + 1], 64, c["dims"].eps))[0]
        want[0, pg, 1, 0, p % page] = Q.pack(v[t])
    got = pool.data.cpu().numpy()
    assert (got == want).all(), np.argwhere(got != want)[:8]
    held = q35.pages_read(pool, 0, i32(c["table"]), i32([0] * T), i32(range(5, 5 + T)))
    assert held.dtype is torch.float16 and held.shape == (T, 2, 1, HD)
    np.testing.assert_array_equal(held[:, 1, 0].cpu().numpy().astype(np.float64), Q.unpack(Q.pack(v)))
    # the bound that the layout promises: half a scale, where nothing is cut and all is finite
    y, w = v.reshape(-1, 32).astype(np.float64), held[:, 1, 0].cpu().numpy().astype(np.float64).reshape(-1, 32)
    ok = (np.abs(y) <= 32768).all(1)
    s = np.maximum((np.maximum(y.max(1), 0) - np.minimum(y.min(1), 0)) / 15 * (1 + 2.0 ** -6), 2.0 ** -20 + (y.max(1) - y.min(1)) / 15)
    assert (np.abs(y - w)[ok].max(1) <= s[ok] / 2).all()
    pool.check()


@pytest.mark.parametrize("fill", [0xFF, 0x7F, 0x00])
def test_what_no_token_occupies_reaches_nothing(fill):
    """Bytes whose words are NaN or large scales behind the sequences' ends and in other pages."""
    c = make(5, 32, 8, 2, [(1, 40), (3, 30), (40, 21), (1, 0)], fill=fill)
    check(c, *run(c))


@pytest.mark.parametrize("sigma", [1e-4, 30.0, 5000.0])
@pytest.mark.parametrize("n", [1, 40])
def test_values_of_any_size(sigma, n):
    c = make(32, 32, 8, 2, [(n, 200)])
    r = np.random.default_rng(3)
    c["pool"][:, :, 1] = Q.pack(sigma * r.standard_normal(c["pool"][:, :, 1].shape[:-1] + (HD,)))
    c["v"] *= np.float32(sigma)
    check(c, *run(c))


def test_large_scores_and_uneven_values():
    c = make(8, 32, 8, 2, [(1, 300), (20, 100)])
    c["qw"] = c["qw"] * 20
    r = np.random.default_rng(1)
    shape = c["pool"].shape[1], c["pool"].shape[3], c["pool"].shape[4]
    c["pool"][0, :, 1] = Q.pack(r.standard_normal(shape + (HD,)) * 10.0 ** r.uniform(-1.5, 1.5, shape + (1,)))
    check(c, *run(c))


def test_shared_pages_layers_and_odd_rotary():
    c = make(6, 16, 8, 2, [(1, 50), (4, 33), (30, 40)], layers=3, layer=2, shared=2, rot=22)
    check(c, *run(c))


def test_stream_larger_than_the_last_level_cache():
    """520000 tokens of two heads, 300 MB: the loads that pass the caches by, and offsets near the end of a pool, against
    parts of the context attended to by themselves and joined in f64."""
    ctx, page, parts = 520000, 64, 8
    dims = q35.dims_2b()
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    n = ctx // page + 1
    pool = q35.PagePool.empty(1, n, page=page, dtype=q35.Q4)
    pool.data.random_(0, 256, generator=g)
    words = pool.data.view(torch.int16)[..., HD // 4:]
    words.copy_(0x3000 + 16 * torch.randint(0, 64, words.shape, generator=g, device="cuda") + 7)  # scales 1/8 .. 1/4, zeros 7
    table = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().cuda()[None]
    qg, k, v = (torch.randn(1, w, generator=g, device="cuda") for w in (4096, 512, 512))
    qw, kw = torch.full((HD,), 0.5, device="cuda"), torch.zeros(HD, device="cuda")
    cos, sin = torch.ones(ctx + 1, 64, device="cuda"), torch.zeros(ctx + 1, 64, device="cuda")
    out = q35.attention_core_paged(dims, pool, 0, qg, k, v, i32([0, 1]), i32([ctx]), table, qw, kw, cos, sin, check=True)
    q = qg.view(8, 2, HD)[:, 0].double()
    q = q / (q.square().mean(-1, keepdim=True) + dims.eps).sqrt() * 1.5
    num, den = torch.zeros(8, HD, dtype=torch.float64, device="cuda"), torch.zeros(8, dtype=torch.float64, device="cuda")
    big = 0.0
    for part in torch.arange(ctx + 1, dtype=torch.int32, device="cuda").chunk(parts):
        kv = q35.pages_read(pool, 0, table, torch.zeros_like(part), part).double()
        for h in range(8):
            s = kv[:, 0, h // 4] @ q[h] / 16.0
            big = max(big, float(s.abs().max()))
            e = (s - 40.0).exp()
            num[h] += e @ kv[:, 1, h // 4]
            den[h] += e.sum()
    want = (num / den[:, None] * torch.sigmoid(qg.view(8, 2, HD)[:, 1].double())).view(1, -1)
    # tests/paged_ref.py's bound; values are at most 8 / 4
    torch.testing.assert_close(out.double(), want, rtol=0, atol=4 * (big + 2) * 2.0 ** -20 * 2.0)


def test_same_bits_on_every_run_and_rows_behind_the_last():
    c = make(37, 16, 8, 2, [(1, 700), (90, 333), (5, 100), (1, 0)])
    T = c["start"][-1]
    for name in ("qg", "k", "v"):
        c[name] = np.concatenate([c[name], np.full((3, c[name].shape[1]), np.nan, np.float32)])
    first = torch.full((T + 3, 2048), 7.0, device="cuda")
    run(c, out=first)
    assert (first[T:] == 7.0).all()
    for _ in range(3):
        again = torch.full((T + 3, 2048), 7.0, device="cuda")
        run(c, out=again)
        assert torch.equal(again, first)


def test_bad_positions_and_pages_are_reported():
    c = make(12, 32, 8, 2, [(2, 40), (3, 50), (1, 20)])
    ok = run(c)[0].clone()
    got, pool = run(dict(c, pos=[40, 10 ** 6, 20]), out=torch.full(ok.shape, 5.0, device="cuda"))
    assert torch.equal(got[:2], ok[:2]) and torch.equal(got[5:], ok[5:]) and (got[2:5] == 5.0).all()
    with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
        pool.check()
    for value in (-1, 10 ** 6):
        table = [list(r) for r in c["table"]]
        table[1][0] = table[1][1] = value
        got, pool = run(dict(c, table=table))
        assert torch.equal(got[:2], ok[:2]) and torch.equal(got[5:], ok[5:])
        with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
            pool.check()


def test_captured_and_replayed():
    """A graph of a step, replayed with other inputs between eager work."""
    c = make(14, 32, 8, 2, [(1, 100), (4, 60), (30, 10)])
    pool = q35.PagePool(d(c["pool"]))
    qg, k, v = d(c["qg"]), d(c["k"]), d(c["v"])
    args = [i32(c["start"]), i32(c["pos"]), i32(c["table"]), d(c["qw"]), d(c["kw"]), d(c["cos"]), d(c["sin"])]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q35.attention_core_paged(c["dims"], pool, 0, qg, k, v, *args)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = q35.attention_core_paged(c["dims"], pool, 0, qg, k, v, *args)
    for seed in range(3):
        r = np.random.default_rng(seed)
        for name, t in (("qg", qg), ("k", k), ("v", v)):
            c[name] = r.standard_normal(c[name].shape).astype(np.float32)
            t.copy_(torch.from_numpy(c[name]))
        pool.data.copy_(torch.from_numpy(c["pool"]))
        graph.replay()
        torch.cuda.synchronize()
        check(c, out, pool)
        eager, _ = run(c)
        assert torch.equal(eager, out)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "q4"])
def test_pages_read(dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    if dtype == "q4":
        data = torch.randint(0, 256, (3, 9, 2, 3, 16, ROW), generator=g, device="cuda", dtype=torch.uint8)
        data.view(torch.int16)[..., HD // 4:] &= 0x77FF  # finite scales
        data.view(torch.int16)[0, 0, 0, 0, 0, HD // 4] = 0x7FF0
        values = torch.from_numpy(Q.unpack(data.cpu().numpy())).half()
    else:
        data = torch.randn((3, 9, 2, 3, 16, HD), generator=g, device="cuda").to(R.TORCH[dtype])
        values = data.cpu()
    pool = q35.PagePool(data)
    table = [[4, 0, 7, -1], [8, 8, -1, 20], [1, 2, 3, 5]]
    rows, pos = [0, 0, 2, 1, 2, 0, 1], [0, 47, 63, 17, 5, 16, 3]
    got = q35.pages_read(pool, 1, i32(table), i32(rows), i32(pos), check=True).cpu()
    for i, (r, p) in enumerate(zip(rows, pos)):
        want = values[1, table[r][p // 16], :, :, p % 16]
        assert torch.equal(got[i], want) and got[i].dtype is values.dtype
    first = q35.pages_read(pool, 0, i32([[0]]), i32([0]), i32([0])).cpu()
    torch.testing.assert_close(first[0], values[0, 0, :, :, 0], rtol=0, atol=0, equal_nan=True)
    for r, p in ((3, 0), (-1, 0), (0, 48), (0, 64), (0, -1), (1, 50)):
        got = q35.pages_read(pool, 1, i32(table), i32([r, 2]), i32([p, 5])).cpu()
        assert (got[0] == 0).all() and torch.equal(got[1], values[1, 1, :, :, 5])
        with pytest.raises(q35.Q35Error, match="Q35_E_RANGE"):
            pool.check()
    assert q35.pages_read(pool, 0, i32(table), i32([]), i32([])).shape == (0, 2, 3, HD)


@pytest.mark.parametrize("page,kv,n", [(16, 1, 3), (16, 3, 40), (64, 2, 300), (256, 1, 5)])
def test_pages_copy(page, kv, n):
    """Pages of 4608 bytes and more, few of them whole units of a block's copy."""
    r = np.random.default_rng(n)
    pages = 2 * n + 7
    data = torch.from_numpy(r.integers(0, 256, (2, pages, 2, kv, page, ROW), dtype=np.uint8))
    pool = q35.PagePool(data.cuda())
    ids = r.permutation(pages)
    src, dst = ids[:n], ids[n:2 * n]
    q35.pages_copy(pool, i32(src), i32(dst), check=True)
    want = data.clone()
    want[:, dst] = data[:, src]
    assert torch.equal(pool.data.cpu(), want)
    other = q35.PagePool(torch.zeros((2, n + 1, 2, kv, page, ROW), dtype=torch.uint8, device="cuda"))
    q35.pages_copy(pool, i32(src), i32(np.arange(n)), to=other, check=True)
    assert torch.equal(other.data.cpu()[:, :n], want[:, src]) and not other.data[:, n].any()
    with pytest.raises(q35.Q35Error, match="Q35_E_SHAPE"):
        q35.pages_copy(pool, i32(src), i32(dst), to=q35.PagePool.empty(2, n, kv, page, dtype=torch.float16))


@pytest.mark.parametrize("page,kv,seqs,out", [(16, 2, 4, 9), (64, 3, 6, 70), (32, 1, 3, 300)])
def test_pages_fork_and_compact(page, kv, seqs, out):
    r = np.random.default_rng(out)
    lens = [int(x) for x in r.integers(0, 5 * page, seqs)]
    parents = [int(x) for x in r.integers(-1, seqs, out)]
    width, grow = 9, [int(x) for x in r.integers(0, 2 * page, out)]
    n_pages = seqs * 6 + out * 4
    ids, table, at = r.permutation(n_pages).tolist(), [], 0
    for n in lens:
        k = -(-n // page)
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    data = torch.from_numpy(r.integers(0, 256, (2, n_pages, 2, kv, page, ROW), dtype=np.uint8))
    pool = q35.PagePool(data.cuda())
    f = q35.pages_fork(pool, i32(table), i32(lens), i32(parents), i32(grow), check=True)
    rows, out_len, refs, copies, short = R.fork(table, lens, parents, grow, n_pages, page)
    assert not short and f.table.tolist() == rows and f.lens.tolist() == out_len and f.refs.tolist() == refs
    want = data.clone()
    for s, t, tokens in copies:
        want[:, t, :, :, :tokens] = data[:, s, :, :, :tokens]
    assert torch.equal(pool.data.cpu(), want)
    c = q35.pages_compact(pool, f.table, check=True)
    rows, refs, used, moves = R.compact(rows, n_pages)
    assert c.table.tolist() == rows and c.refs.tolist() == refs and c.used.tolist() == [used]
    after = want.clone()
    for s, t in moves:
        after[:, t] = want[:, s]
    assert torch.equal(pool.data.cpu(), after)


def test_pool_of_another_shape_is_refused():
    with pytest.raises(AssertionError):
        q35.PagePool(torch.zeros((1, 4, 2, 2, 16, 256), dtype=torch.uint8, device="cuda"))
    assert q35.PagePool.empty(1, 2, 3, 16, dtype=q35.Q4).data.shape == (1, 2, 2, 3, 16, ROW)
    with pytest.raises(AssertionError):
        q35.PagePool.empty(1, 2, head_dim=128, dtype=q35.Q4)


def test_pages_beyond_32bit_offsets():
    """A small case in the last pages of the second of two layers, 2.2 GB each."""
    seqs = [(1, 300), (5, 70), (200, 130)]
    c = make(12, 64, 8, 2, seqs)
    small = d(c["pool"])
    used, n = small.shape[1], 60000
    pool = q35.PagePool.empty(2, n, page=64, dtype=q35.Q4)
    assert pool.data[1, n - used:].data_ptr() - pool.data.data_ptr() > 2 ** 32
    pool.data[1, n - used:] = small[0]
    high = [[p + n - used if p >= 0 else -1 for p in row] for row in c["table"]]
    out, _ = run(dict(c, layer=1, table=high), pool)
    check(c, out, q35.PagePool(pool.data[1:, n - used:].clone()))
    pool.check()
    last = [(b, x + y - 1) for b, (x, y) in enumerate(seqs)]
    rows, at = i32([b for b, _ in last]), i32([p for _, p in last])
    got = q35.pages_read(pool, 1, i32(high), rows, at, check=True)
    want = pool.data[1, n - used:]
    for i, (b, p) in enumerate(last):
        assert torch.equal(got[i].cpu(), torch.from_numpy(Q.unpack(want[c["table"][b][p // 64], :, :, p % 64].cpu().numpy())).half())
    want = want[-2:].clone()
    q35.pages_copy(pool, i32([n - 2, n - 1]), i32([0, 1]), check=True)
    assert torch.equal(pool.data[1, :2], want)
    pool.data[1, -2:] = 0
    q35.pages_copy(pool, i32([0, 1]), i32([n - 2, n - 1]), check=True)
    assert torch.equal(pool.data[1, -2:], want)


@pytest.mark.parametrize("heads,kv,seqs", [
    (8, 2, [(5, 700 + 60 * i) for i in range(12)]),               # two tiles each; a block's share is a part of one
    (8, 2, [(1, 3000 + 130 * (i % 9)) for i in range(20)]),
    (4, 1, [(1, 31 + 32 * (i % 5)) for i in range(200)] + [(1, 9000)]),
    (4, 2, [(1, (37 * i) % 211) for i in range(300)]),            # more tiles than blocks
    (4, 1, [(1, (53 * i) % 150) for i in range(257)]),            # as many as a thread of the plan each, and one
    (16, 1, [(2, 5000), (1, 70), (2, 1)]),
    (4, 1, [(1, 1500 if i % 2 else 2) for i in range(180)]),      # whole parts come out too uneven
])
def test_division_of_the_work(heads, kv, seqs):
    c = make(len(seqs), 64, heads, kv, seqs)
    check(c, *run(c))


@pytest.mark.parametrize("rise", [0.05, 0.5, 0.55, 4.0, -0.5])
def test_scores_that_rise_along_the_context(rise):
    """The running maximum is passed by little or much in every step (a step of 128 tokens rises by 23 rise / 4 powers of two)."""
    c = make(3, 64, 8, 2, [(1, 511), (3, 400)])
    r = np.random.default_rng(8)
    u = r.standard_normal(HD)
    c["qg"].reshape(4, 8, 2, HD)[:, :, 0] = u
    c["qw"][:], c["cos"][:], c["sin"][:] = 0.0, 1.0, 0.0
    for b, (n, ctx) in enumerate([(1, 511), (3, 400)]):
        for t in range(ctx):
            c["pool"][0, c["table"][b][t // 64], 0, :, t % 64] = Q.pack(u * (rise * t / 512))
    check(c, *run(c))


@pytest.mark.parametrize("page,heads,kv,seqs", [c for c in CASES if max(n for n, _ in c[3]) * c[1] // c[2] > 32])
def test_chunks_beside_few_tokens(page, heads, kv, seqs):
    """Batches under tables and rotary rows for contexts so long that a chunk is not taken for few tokens."""
    T = sum(n for n, _ in seqs)
    cap = 350000 * 16 // 9 // (-(-T * heads // kv // 16) * kv) + 2 * page
    c = make(len(seqs) + T, page, heads, kv, seqs)
    c["table"] = [row + [-1] * (cap // page + 1 - len(row)) for row in c["table"]]
    c["cos"], c["sin"] = (np.concatenate([x, np.zeros((cap - len(x), x.shape[1]), np.float32)]) for x in (c["cos"], c["sin"]))
    check(c, *run(c))


@pytest.mark.parametrize("heads,kv,seqs", [
    (8, 2, [(500, 0), (500, 0)]),                                 # as many tiles as blocks, of 1 to 16 units
    (8, 2, [(500, 0), (510, 0)]),                                 # one more than blocks
    (8, 2, [(31, 200)] * 8 + [(120, 3)]),
    (16, 1, [(128, 0)] * 4),
    (4, 4, [(64, 700), (33, 0), (1, 0)]),
    (8, 2, [(1000, 20)]),
    (16, 1, [(9, 400)]),
])
def test_prompts_as_few_tokens(heads, kv, seqs):
    c = make(sum(n for n, _ in seqs), 64, heads, kv, seqs)
    check(c, *run(c))


@pytest.mark.parametrize("heads,kv,seqs", [
    (8, 2, [(1, 9000), (0, 5)]),                                  # 71 parts of a step of each wave
    (8, 2, [(1, 700), (1, 3), (1, 64), (1, 2000), (3, 2500)]),
    (4, 4, [(2, 900)] * 3),
    (16, 1, [(1, 4097)]),
    (4, 1, [(1, 2)] * 500 + [(1, 5000)]),
])
def test_parts_of_a_tile(heads, kv, seqs):
    c = make(len(seqs), 64, heads, kv, seqs)
    check(c, *run(c))

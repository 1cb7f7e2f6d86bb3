"""Forks of tables whose rows share pages that are not full: a page with room stands in one row afterwards, once."""
import numpy as np
import pytest
import torch

import paged_ref as R
import q35

HD = 256


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def fork(table, lens, parents, grow, n_pages, page):
    """(table_out, lens_out, refs, copies [(row, entry, source, tokens)]) by the definition; enough free pages."""
    width = len(table[0])
    out_len = [lens[p] if p >= 0 else 0 for p in parents]
    rows = [list(table[p][:n // page]) if p >= 0 else [] for p, n in zip(parents, out_len)]
    named = {e for r in rows for e in r}
    copies = []
    for j, (p, n) in enumerate(zip(parents, out_len)):
        if n % page:
            e = table[p][n // page]
            if e not in named:  # neither full in a row nor kept by a row before
                named.add(e)
                rows[j].append(e)
            else:
                copies.append((j, n // page, e, n % page))
    free = iter(e for e in range(n_pages) if e not in named)
    for r, n, g in zip(rows, out_len, grow or [0] * len(parents)):
        r += [next(free) for _ in range(-(-(n + g) // page) - len(r))]
        r += [-1] * (width - len(r))
    refs = np.bincount([e for r in rows for e in r if e >= 0], minlength=n_pages).tolist()
    return rows, out_len, refs, copies


def test_definition_of_tables_without_shared_room():
    """Where no page with room is shared, it is the definition that the other tests use."""
    r = np.random.default_rng(0)
    for _ in range(50):
        page, seqs = 16, int(r.integers(1, 6))
        lens = [int(n) for n in r.integers(0, 60, seqs)]
        ids = r.permutation(60).tolist()
        table = [[ids.pop() for _ in range(-(-n // page))] for n in lens]
        table = [t + [-1] * (7 - len(t)) for t in table]
        parents = [int(p) for p in r.integers(-1, seqs, 8)]
        grow = [int(g) for g in r.integers(0, 30, 8)]
        rows, out_len, refs, copies = fork(table, lens, parents, grow, 60, page)
        want = R.fork(table, lens, parents, grow, 60, page)
        assert (rows, out_len, refs) == want[:3] and [(s, rows[j][at], t) for j, at, s, t in copies] == want[3]


def check(n_pages, page, layers, kv, table, lens, parents, grow, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    data = torch.randn((layers, n_pages, 2, kv, page, HD), generator=g, device="cuda").bfloat16()
    pool = q35.PagePool(data.clone())
    f = q35.pages_fork(pool, i32(table), i32(lens), i32(parents), i32(grow), check=True)
    rows, out_len, refs, copies = fork(table, lens, parents, grow, n_pages, page)
    assert f.table.cpu().tolist() == rows
    assert f.lens.cpu().tolist() == out_len and f.refs.cpu().tolist() == refs
    # pages with room: one row, once
    for row, n in zip(rows, out_len):
        if n % page:
            assert refs[row[n // page]] == 1
    for j, at, s, t in copies:
        data[:, rows[j][at], :, :, :t] = data[:, s, :, :, :t].clone()
    assert torch.equal(pool.data, data)
    return f, pool


# one launch; two (many copies); counts in memory (more pages than LDS counts)
POOLS = [(40, 1, 1), (40, 6, 16), (17000, 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("n_pages,layers,kv", POOLS)
@pytest.mark.parametrize("table,lens,parents,grow", [
    ([[4, -1, -1], [4, 2, -1]], [8, 20], [0, 1], [4, 1]),            # cut back into a prefix that the other one holds
    ([[4, -1, -1], [4, 2, -1]], [8, 20], [1, 0, 0], [1, 4, 0]),
    ([[4, 3, -1], [4, 3, -1]], [20, 20], [0, 1], [1, 1]),            # one partly filled page in two rows
    ([[4, 3, -1], [4, 3, -1], [4, 3, -1]], [20, 25, 17], [2, 2, 0, 1, -1, 1], [1, 9, 12, 0, 3, 1]),
    ([[7, 7, -1], [7, -1, -1]], [20, 5], [1, 0], [2, 2]),            # one row that names a page twice
    ([[5, 6, 1], [5, 6, 1], [6, 1, 0]], [48, 33, 40], [1, 0, 2], [1, 0, 8]),
], ids=["prefix", "prefix-forked", "same-page", "same-page-forked", "twice", "full-elsewhere"])
def test_fork_of_shared_pages_with_room(n_pages, layers, kv, table, lens, parents, grow):
    print(n_pages, layers, kv, table, lens, parents, flush=True)
    check(n_pages, 16, layers, kv, table, lens, parents, grow)


@pytest.mark.gpu
@pytest.mark.parametrize("n_pages,layers,kv", [(300, 1, 1), (300, 6, 4), (16500, 2, 1)])
@pytest.mark.parametrize("seed", range(4))
def test_fork_of_random_shared_tables(n_pages, layers, kv, seed):
    """Tables of few pages, so that rows share them in every way."""
    r = np.random.default_rng(seed)
    seqs, out, page, width = int(r.integers(2, 60)), int(r.integers(2, 90)), 16, 6
    few = [3, 9, 25, 60][seed]
    lens = [int(n) for n in r.integers(0, 4 * page, seqs)]
    table = [[int(e) for e in r.integers(0, few, -(-n // page))] for n in lens]
    table = [t + [-1] * (width - len(t)) for t in table]
    parents = [int(p) for p in r.integers(-1, seqs, out)]
    check(n_pages, page, layers, kv, table, lens, parents, [int(g) for g in r.integers(0, page, out)], seed)


@pytest.mark.gpu
def test_fork_of_one_prompt_in_many_rows():
    """More rows than threads name one partly filled page."""
    rows = 1500
    check(1700, 16, 1, 1, [[4, 3, -1, -1]] * rows, [16 + 1 + i % 15 for i in range(rows)], list(range(rows)), [i % 3 for i in range(rows)])


@pytest.mark.gpu
def test_sequences_of_a_shared_prefix_do_not_meet():
    """A sequence cut back into a prefix that another one holds, forked with room and appended to: the other's
    outputs and context are those of its own cache alone."""
    page, dims = 16, q35.dims_2b()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    pool = q35.PagePool(rnd(1, 12, 2, 2, page, HD))
    qg, k, v, qw, kw = rnd(5, 4096), rnd(5, 512), rnd(5, 512), rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    cos, sin = (torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, 64))
    alone = q35.PagePool(pool.data.clone())
    want = q35.attention_core_paged(dims, alone, 0, qg[4:], k[4:], v[4:], i32([0, 1]), i32([20]), i32([[4, 2, -1]]), qw, kw, cos, sin)
    f = q35.pages_fork(pool, i32([[4, -1, -1], [4, 2, -1]]), i32([8, 20]), i32([0, 1]), i32([4, 1]))
    got = q35.attention_core_paged(dims, pool, 0, qg, k, v, i32([0, 4, 5]), f.lens, f.table, qw, kw, cos, sin, check=True)
    # (the same sequence, tile and order of sums in both calls)
    assert torch.equal(got[4:], want)
    assert torch.equal(pool.data[:, 4], alone.data[:, 4])

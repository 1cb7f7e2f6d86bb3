"""Beam search as a program runs it: BatchDecoder.beam_search against the same search that starts every step's
hypotheses from nothing, and the operators together over a cache in 4 bits and DeltaNet states."""
import numpy as np
import pytest
import torch

import beam_ref as B
import q35

pytestmark = pytest.mark.gpu

HD = 256


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def hybrid_dims():
    return q35.make_dims(hidden=512, ffn=1536, vocab=8192, n_layers=4, lin_heads=4, attn_heads=4, kv_heads=2)


def reference(bt, prompts, beams, n_new, stop_ids=()):
    """[(ids, sum of log probabilities)] per prompt: every step feeds all hypotheses whole."""
    G, V = len(prompts), bt.model.dims.vocab
    hyps = [[np.asarray(p, np.int32)] * beams for p in prompts]
    scores = np.full((G, beams), -np.inf, np.float32)
    scores[:, 0] = 0.0
    ended = np.full(G * beams, -1)
    count = np.zeros(G * beams, int)
    for i in range(n_new):
        bt.reset()
        bt.generate([h for g in hyps for h in g], 0, prefill=True)
        x = bt.tensor("logits", np.float32).reshape(G * beams, V).astype(np.float64)
        (s, p, t), _ = B.select(x, scores, beams, ended)
        rows = [h for g in hyps for h in g]
        hyps = [[np.append(rows[p[g, w]], t[g, w]).astype(np.int32) for w in range(beams)] for g in range(G)]
        old, scores = ended.copy(), s.astype(np.float32)
        new_count, new_ended = count.copy(), ended.copy()
        for r, (pa, tk) in enumerate(zip(p.ravel(), t.ravel())):
            over = old[pa] >= 0
            new_count[r] = count[pa] if over else i + 1
            new_ended[r] = tk if over or tk in stop_ids else -1
        count, ended = new_count, new_ended
    return [[(hyps[g][w][len(prompts[g]):][:count[g * beams + w]], float(scores[g, w])) for w in range(beams)] for g in range(G)]


def same(got, want, penalty=0.0):
    for g, w in zip(got, want):
        w = sorted([(ids, s / len(ids) ** penalty) for ids, s in w], key=lambda h: -h[1])
        assert len(g) == len(w)
        for (a, sa), (b, sb) in zip(g, w):
            np.testing.assert_array_equal(a, b)
            # sums of up to 7 log probabilities of logits that are 1e-5 apart (test_gpu_batch's bound, relative) and of size 10
            assert abs(sa - sb) < 7 * 1e-4, (sa, sb)


@pytest.mark.parametrize("mode", ["graph", "stream"])
def test_beam_search_matches_whole_hypotheses(mode):
    d = hybrid_dims()
    m = q35.TextForCausalLM(d, seed=3, tmax=64)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, d.vocab, n).astype(np.int32) for n in (9, 1, 17)]
    bt = q35.BatchDecoder(m, 9, 40)
    want = reference(bt, prompts, 3, 7)
    same(bt.beam_search(prompts, 3, 7, mode=mode), want)
    np.testing.assert_array_equal(bt.positions(), np.repeat([len(p) + 6 for p in prompts], 3))
    # an id that some hypotheses hold ends them
    stop = int(want[0][0][0][2])
    ended = reference(bt, prompts, 3, 7, (stop,))
    assert any(len(ids) < 7 for ids, _ in ended[0])
    same(bt.beam_search(prompts, 3, 7, stop_ids=[stop], mode=mode), ended)
    same(bt.beam_search(prompts, 3, 7, stop_ids=[stop], length_penalty=1.0, mode=mode), ended, 1.0)
    bt.close()
    m.close()


def test_one_beam_is_greedy_and_an_early_end():
    d = hybrid_dims()
    m = q35.TextForCausalLM(d, seed=3, tmax=80)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, d.vocab, 6).astype(np.int32) for _ in range(2)]
    bt = q35.BatchDecoder(m, 2, 70)
    toks, _ = bt.generate(prompts, 39, prefill=True)
    got = bt.beam_search(prompts, 1, 40)
    for g in range(2):
        np.testing.assert_array_equal(got[g][0][0], toks[g])
    stop = sorted({int(t) for t in toks[:, :8].ravel()})
    got = bt.beam_search(prompts, 1, 40, stop_ids=stop)
    assert bt.positions().max() < 6 + 39  # (both ended at once: the search saw it after 16 steps)
    assert [len(g[0][0]) for g in got] == [1, 1] and got[0][0][0][0] == toks[0, 0]
    bt.close()
    m.close()


def test_forks_of_rows_at_other_positions_are_refused():
    d = hybrid_dims()
    m = q35.TextForCausalLM(d, seed=4, tmax=40)
    rng = np.random.default_rng(1)
    bt = q35.BatchDecoder(m, 4, 30)
    bt.generate([rng.integers(0, d.vocab, n).astype(np.int32) for n in (5, 5, 8, 8)], 0, prefill=True)
    name = "layers.0.linear_attn.recurrent_state"
    before = bt.tensor(name, np.float32).reshape(4, -1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    bt.fork(i32([1, 2, -1, 2]), i32([3, 8191, -1, 9000]), status=status)
    torch.cuda.synchronize()
    after = bt.tensor(name, np.float32).reshape(4, -1)
    for j, p in enumerate([1, 1, 2, 2]):  # row 1 asked for a row at another position
        np.testing.assert_array_equal(after[j], before[p])
    assert bt.tensor("token", np.int32).tolist() == [3, 8191, 0, 0] and int(status) == q35._lib.Q35_STATUS_ARG
    hist = bt.tensor("hist", np.int32).reshape(4, 30)
    assert [hist[j, n - 1] for j, n in enumerate((5, 5, 8, 8))] == [3, 8191, 0, 0]
    status.zero_()
    torch.cuda.synchronize()
    bt.fork(i32([1, 0, 3, -1]), i32([1, 2, 3, -1]), status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    with pytest.raises(AssertionError):
        bt.fork(i32([0, 1]))
    bt.close()
    m.close()


def test_operators_together():
    """Steps of a beam search over a pool in 4 bits and a DeltaNet core's states - pages_fork, attention, the core,
    beam_select, states_fork - against hypotheses computed from nothing, with beams that end on the way."""
    dims = q35.dims_2b()
    page, G, W, V, steps, T0, heads = 16, 2, 4, 600, 10, 37, 4
    R = G * W
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    emb, wq, wk, wv = rnd(V, 64), rnd(64, 4096, f=0.125), rnd(64, 512, f=0.125), rnd(64, 512, f=0.125)
    wm, wb, conv_w = rnd(64, heads * 384, f=0.125), rnd(64, 2 * heads, f=0.125), rnd(heads * 384, 4, f=0.5)
    head = rnd(2048 + heads * 128, V, f=0.1)
    qw, kw = rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    cos, sin = (torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, 128))
    prompts = torch.randint(0, V, (G, T0), generator=g, device="cuda")
    stop = 7

    def core(tok, conv, rec):
        e = emb[tok]
        bg = e @ wb
        bg = torch.cat([torch.sigmoid(bg[:, :heads]), -torch.nn.functional.softplus(bg[:, heads:])], 1).contiguous()
        return q35.gated_delta_rule_decode((e @ wm).contiguous(), bg, conv, conv_w, rec, heads)

    def states(n):
        return [torch.zeros(n, heads * 384, 3, device="cuda"), torch.zeros(n, heads, 128, 128, device="cuda")]

    def attend(pool, tok, start, lens, table):
        e = emb[tok]
        return q35.attention_core_paged(dims, pool, 0, e @ wq, e @ wk, e @ wv, start, lens, table, qw, kw, cos, sin)

    # the search
    pool = q35.PagePool.empty(1, 80, page=page, dtype=q35.Q4)
    pool.data.fill_(0xFF)
    f = q35.pages_fork(pool, i32([[-1] * 5]), i32([0]), i32([-1] * G), i32([T0] * G))
    out = attend(pool, prompts.flatten(), i32([T0 * i for i in range(G + 1)]), f.lens, f.table)[T0 - 1::T0]
    st = states(G)
    for t in range(T0):
        o = core(prompts[:, t].contiguous(), *st)
    logits = torch.cat([out, o], 1).repeat_interleave(W, 0) @ head
    scores = torch.full((G, W), -float("inf"), device="cuda")
    scores[:, 0] = 0.0
    r = q35.beam_select(logits, scores, W, check=True)
    parents = r.parents
    table, lens = f.table, torch.full((G,), T0, dtype=torch.int32, device="cuda")
    row_of = torch.div(parents.view(-1), W, rounding_mode="floor").int()  # (one sequence per prompt so far)
    wide = states(R)
    st = q35.states_fork(st, row_of, out=wide, check=True)
    seqs = [[int(t)] for t in r.tokens.view(-1)]
    ended = torch.where(r.tokens.view(-1) == stop, r.tokens.view(-1), -1)
    fork_parents = row_of
    start = i32(range(R + 1))
    for _ in range(steps):
        f = q35.pages_fork(pool, table, lens, fork_parents, i32([1] * R), check=True)
        table, lens = f.table, f.lens
        tok = r.tokens.view(-1)
        out = attend(pool, tok, start, lens, table)
        lens = lens + 1
        o = core(tok, *st)
        r = q35.beam_select(torch.cat([out, o], 1) @ head, r.scores, W, ended=ended, check=True)
        fork_parents = r.parents.view(-1).contiguous()
        q35.states_fork(st, fork_parents, check=True)
        over = ended[fork_parents.long()]
        t = r.tokens.view(-1)
        ended = torch.where((over >= 0) | (t == stop), t, -1)
        seqs = [seqs[int(p)] + [int(x)] for p, x in zip(fork_parents, t)]
    pool.check()

    # from nothing
    def forward(hyps):  # [(prompt, ids)] of one length
        n = T0 + len(hyps[0][1])
        ids = torch.stack([torch.cat([prompts[p], torch.tensor(s, device="cuda", dtype=prompts.dtype)]) for p, s in hyps])
        own = q35.PagePool.empty(1, 5 * len(hyps), page=page, dtype=q35.Q4)
        out = attend(own, ids.flatten(), i32([n * i for i in range(len(hyps) + 1)]), i32([0] * len(hyps)),
                     i32(np.arange(5 * len(hyps)).reshape(-1, 5)))[n - 1::n]
        s = states(len(hyps))
        for t in range(n):
            o = core(ids[:, t].contiguous(), *s)
        return (torch.cat([out, o], 1) @ head).double().cpu().numpy()

    hyps = [(p, []) for p in range(G) for _ in range(W)]
    sc = np.full((G, W), -np.inf, np.float32)
    sc[:, 0] = 0.0
    end = np.full(R, -1)
    for _ in range(steps + 1):
        (s, p, t), _ = B.select(forward(hyps), sc, W, end)
        sc, p, t = s.astype(np.float32), p.ravel(), t.ravel()
        hyps = [(hyps[a][0], hyps[a][1] + [int(b)]) for a, b in zip(p, t)]
        end = np.where((end[p] >= 0) | (t == stop), t, -1)
    assert seqs == [h[1] for h in hyps]
    # 11 sums of f32 logits of size 10 from outputs that are a few 1e-6 apart (chunks and single tokens)
    np.testing.assert_allclose(r.scores.cpu().numpy(), sc, rtol=0, atol=2e-3)


def test_forks_without_a_stream_wait_for_the_tensors():
    """parents and tokens are written late on torch's stream, and overwritten after the call."""
    d = hybrid_dims()
    m = q35.TextForCausalLM(d, seed=4, tmax=40)
    rng = np.random.default_rng(1)
    bt = q35.BatchDecoder(m, 4, 30)
    bt.generate([rng.integers(0, d.vocab, 5).astype(np.int32) for _ in range(4)], 0, prefill=True)
    name = "layers.0.linear_attn.recurrent_state"
    before = bt.tensor(name, np.float32).reshape(4, -1)
    parents, tokens, want, ids = i32([0, 1, 2, 3]), i32([0] * 4), i32([3, 0, 0, 1]), i32([5, 6, 7, 8])
    big = torch.randn(8192, 8192, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    for _ in range(20):
        big = (big @ big).clamp(-1, 1)
    parents.copy_(want)
    tokens.copy_(ids)
    bt.fork(parents, tokens)
    parents.zero_()
    tokens.zero_()
    torch.cuda.synchronize()
    after = bt.tensor(name, np.float32).reshape(4, -1)
    for j, p in enumerate([3, 0, 0, 1]):
        np.testing.assert_array_equal(after[j], before[p])
    assert bt.tensor("token", np.int32).tolist() == [5, 6, 7, 8]
    bt.close()
    m.close()


def test_searches_that_do_not_fit_are_refused():
    m = q35.TextForCausalLM(hybrid_dims(), seed=4, tmax=40)
    bt = q35.BatchDecoder(m, 66, 12)
    for prompts, beams, n_new in (([[1]], 66, 2), ([[1], [2]], 32, 2), ([[1], [2]], 33, 0), ([[1, 2, 3], [2]], 33, 11)):
        with pytest.raises(AssertionError):
            bt.beam_search(prompts, beams, n_new)
    got = bt.beam_search([[1, 2, 3], [2]], 33, 2)
    assert [len(g) for g in got] == [33, 33] and all(len(ids) == 2 for g in got for ids, _ in g)
    bt.close()
    m.close()

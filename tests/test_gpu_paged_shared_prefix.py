"""Paged attention of many samples of one long context: more to read than the last-level cache holds, most of it the same."""
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu

HD = 256


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,seqs,shared,new", [
    (torch.float32, 33, 124, 1), (torch.bfloat16, 64, 70, 1), (torch.float16, 70, 62, 2), (torch.bfloat16, 40, 100, 5),
    (torch.bfloat16, 64, 4, 1),
])
def test_samples_of_one_context(dtype, seqs, shared, new):
    """128 pages of 64 tokens each, the first `shared` of them one set: the same bits as with pages of their own, whichever
    way the cache is read."""
    page, pages, dims = 64, 128, q35.dims_2b()
    g = torch.Generator(device="cuda")
    g.manual_seed(seqs)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    own = pages - shared
    pool = q35.PagePool(rnd(1, shared + seqs * own, 2, 2, page, HD).to(dtype))
    first = torch.arange(shared, device="cuda").expand(seqs, -1)
    table = torch.cat([first, shared + torch.arange(seqs * own, device="cuda").view(seqs, own)], 1).int()
    alone = q35.PagePool(pool.data[:, table.flatten().long()].contiguous())
    T, cached = seqs * new, pages * page - 20
    args = rnd(T, 4096), rnd(T, 512), rnd(T, 512)
    start, pos = i32(*range(0, T + 1, new)), i32(*[cached] * seqs)
    norms = rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    rope = [torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, pages * page)]
    got = q35.attention_core_paged(dims, pool, 0, *args, start, pos, table, *norms, *rope, check=True)
    want = q35.attention_core_paged(dims, alone, 0, *args, start, pos, i32(*range(seqs * pages)).view(seqs, pages), *norms, *rope, check=True)
    assert torch.equal(got, want)
    assert torch.equal(pool.data[:, table.flatten().long()], alone.data)
    if dtype != torch.float32:
        return  # (the contiguous caches are f32)
    kc, vc = (alone.data[0, -pages:, i].permute(1, 0, 2, 3).reshape(2, -1, HD).contiguous() for i in (0, 1))
    last = slice(T - new, T)
    whole = q35.attention_core_prefill(dims, *(a[last].contiguous() for a in args), *norms, kc, vc, cached, *rope)
    # two f32 computations of 8172 weights, each off by what tests/paged_ref.py allows for scores of 12
    torch.testing.assert_close(got[last], whole, rtol=0, atol=2 * 4 * 14 * 2.0 ** -20 * float(vc.abs().max()))

"""Paged attention of batches of fixed slots, most of them empty."""
import numpy as np
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu

HD = 256


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("slots,new,cached,at", [(256, 256, 4000, 100), (64, 64, 9000, 0), (33, 40, 16000, 32)])
def test_one_chunk_among_empty_slots(slots, new, cached, at, dtype):
    """One slot's chunk behind a long context goes the way that it goes alone, to the same bits: not tile by tile of a
    few tokens, each over the whole context."""
    page, dims = 64, q35.dims_2b()
    g = torch.Generator(device="cuda")
    g.manual_seed(slots)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    n = -(-(new + cached) // page)
    pools = [q35.PagePool(rnd(1, n, 2, 2, page, HD).to(dtype))]
    pools.append(q35.PagePool(pools[0].data.clone()))
    row = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().cuda()
    table = torch.full((slots, n), -1, dtype=torch.int32, device="cuda")
    table[at] = row
    args = rnd(new, 4096), rnd(new, 512), rnd(new, 512)
    norms = rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    rope = [torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, new + cached)]
    start, pos = [0] * (at + 1) + [new] * (slots - at), [0] * slots
    pos[at] = cached
    among = q35.attention_core_paged(dims, pools[0], 0, *args, i32(start), i32(pos), table, *norms, *rope, check=True)
    alone = q35.attention_core_paged(dims, pools[1], 0, *args, i32([0, new]), i32([cached]), row[None], *norms, *rope, check=True)
    assert torch.equal(among, alone) and torch.equal(pools[0].data, pools[1].data)


@pytest.mark.parametrize("slots,new,cached", [(40, 20, 60), (33, 33, 700)])
def test_one_short_chunk_among_empty_slots(slots, new, cached):
    """Behind short contexts its tiles may go either way: the outputs are those of the chunk alone but for the order of sums."""
    page, dims = 64, q35.dims_2b()
    g = torch.Generator(device="cuda")
    g.manual_seed(slots)
    rnd = lambda *s, f=1.0: torch.randn(s, generator=g, device="cuda") * f
    n = -(-(new + cached) // page)
    pool = q35.PagePool(rnd(1, n, 2, 2, page, HD))
    table = torch.full((slots, n), -1, dtype=torch.int32, device="cuda")
    table[3] = torch.arange(n, device="cuda")
    args = rnd(new, 4096), rnd(new, 512), rnd(new, 512)
    norms = rnd(HD, f=0.2) + 0.5, rnd(HD, f=0.2)
    rope = [torch.from_numpy(a).cuda() for a in q35.rope_tables(dims, new + cached)]
    pos = [0] * slots
    pos[3] = cached
    among = q35.attention_core_paged(dims, pool, 0, *args, i32([0] * 4 + [new] * (slots - 3)), i32(pos), table, *norms, *rope, check=True)
    alone = q35.attention_core_paged(dims, pool, 0, *args, i32([0, new]), i32([cached]), table[3:4], *norms, *rope, check=True)
    # two f32 computations, each off by what tests/paged_ref.py allows: scores of 12 at the most
    torch.testing.assert_close(among, alone, rtol=0, atol=2 * 4 * 14 * 2.0 ** -20 * float(pool.data.abs().max()))

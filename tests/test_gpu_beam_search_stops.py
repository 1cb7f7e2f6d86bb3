"""Stop ids of a beam search: any iterable, any number of them."""
import warnings

import numpy as np
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def batch():
    d = q35.make_dims(hidden=512, ffn=1536, vocab=8192, n_layers=4, lin_heads=4, attn_heads=4, kv_heads=2)
    m = q35.TextForCausalLM(d, seed=3, tmax=40)
    bt = q35.BatchDecoder(m, 6, 40)
    yield bt
    bt.close()
    m.close()


PROMPTS = [np.arange(100, 109, dtype=np.int32), np.arange(7, dtype=np.int32)]


def same(a, b):
    assert [len(g) for g in a] == [len(g) for g in b]
    for g, h in zip(a, b):
        for (x, s), (y, t) in zip(g, h):
            assert x.tolist() == y.tolist() and s == t


def test_any_iterable(batch):
    free = batch.beam_search(PROMPTS, 3, 8)
    stop = int(free[0][0][0][2])
    want = batch.beam_search(PROMPTS, 3, 8, stop_ids=[stop, 8191])
    assert any(len(ids) < 8 for g in want for ids, _ in g)
    for ids in (iter([stop, 8191]), (t for t in (stop, 8191)), {stop, 8191}, np.array([stop, 8191]), torch.tensor([stop, 8191]), (stop, 8191, stop)):
        same(batch.beam_search(PROMPTS, 3, 8, stop_ids=ids), want)
    same(batch.beam_search(PROMPTS, 3, 8, stop_ids=iter(())), free)


@pytest.mark.parametrize("n", [1, 200])
def test_steps_do_not_synchronise(batch, n):
    """As many waits of the host for a search of 4 steps as for one of 12 (the end that stop ids bring is looked for after 16)."""
    def waits(n_new):
        with warnings.catch_warnings(record=True) as told:
            warnings.simplefilter("always")
            torch.cuda.set_sync_debug_mode("warn")
            try:
                batch.beam_search(PROMPTS, 3, n_new, stop_ids=range(4000, 4000 + n))
            finally:
                torch.cuda.set_sync_debug_mode("default")
        return sum("called a synchronizing" in str(w.message) for w in told)

    waits(1)  # (what is made once)
    few = waits(4)
    assert few > 0 and waits(12) == few

"""Token scores of rows that are sure of a token: no log probability above 0, and 0 where nothing else is open."""
import numpy as np
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 7, 3000, 70001, 248320])
def test_one_open_token(V, dtype):
    x = torch.full((4, V), -float("inf"), device="cuda", dtype=DT[dtype])
    at = [0, V - 1, V // 2, V // 3]
    for m, t in enumerate(at):
        x[m, t] = [3.5, -11.25, 0.0, 700.0][m]
    t = torch.tensor(at, dtype=torch.int32, device="cuda")
    r = q35.token_logprobs(x, t, top=1)
    assert (r.logprob == 0).all() and (r.entropy == 0).all() and (r.rank == 0).all()
    assert r.top_ids.flatten().tolist() == at and (r.top_logprobs == 0).all()


@pytest.mark.parametrize("V", [2, 3000, 248320])
def test_two_open_tokens(V):
    """Gaps of 0 to 40: the sum is 1 + e^-gap, held to half a step of f32 (2^-24) by each of its few sums."""
    gaps = np.linspace(0.0, 40.0, 641).astype(np.float32)
    x = torch.full((len(gaps), V), -float("inf"), device="cuda")
    x[:, V - 1] = 1.5
    x[:, 0] = torch.from_numpy(np.float32(1.5) - gaps).cuda()
    d = 1.5 - x[:, 0].double().cpu().numpy()
    hi = -np.log1p(np.exp(-d))
    for target, want in ((V - 1, hi), (0, hi - d)):
        r = q35.token_logprobs(x, torch.full((len(gaps),), target, dtype=torch.int32, device="cuda"), top=2)
        got = r.logprob.double().cpu().numpy()
        assert (got <= 0).all() and (r.top_logprobs <= 0).all() and (r.entropy >= 0).all()
        assert (np.abs(got - want) <= 2.0 ** -22 + 2.0 ** -23 * np.abs(want)).all(), np.abs(got - want).max()


def test_peaked_rows_of_a_vocabulary():
    """Rows whose highest token has nearly all of the weight."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn((64, 50257), generator=g, device="cuda")
    t = torch.arange(64, device="cuda") * 700
    x[torch.arange(64, device="cuda"), t] = torch.linspace(5.0, 60.0, 64, device="cuda")
    r = q35.token_logprobs(x, t.int(), top=3)
    want = torch.log_softmax(x.double(), 1).gather(1, t[:, None])[:, 0]
    assert (r.logprob <= 0).all() and (r.top_logprobs <= 0).all()
    assert ((r.logprob.double() - want).abs() <= 2.0 ** -21 + 2.0 ** -23 * want.abs()).all()

"""BatchDecoder.fork on torch's default stream, whose handle is 0."""
import numpy as np
import pytest
import torch

import q35

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


@pytest.mark.parametrize("own", [True, False])
def test_forks_wait_for_late_tensors(own):
    """parents and tokens are written late on torch's stream, and overwritten after the call: with handle 0, and on a stream
    that the steps and the tensors share."""
    d = q35.make_dims(hidden=512, ffn=1536, vocab=8192, n_layers=4, lin_heads=4, attn_heads=4, kv_heads=2)
    m = q35.TextForCausalLM(d, seed=4, tmax=40)
    rng = np.random.default_rng(1)
    bt = q35.BatchDecoder(m, 4, 30)
    bt.generate([rng.integers(0, d.vocab, 5).astype(np.int32) for _ in range(4)], 0, prefill=True)
    name = "layers.0.linear_attn.recurrent_state"
    before = bt.tensor(name, np.float32).reshape(4, -1)
    parents, tokens, want, ids = i32([0, 1, 2, 3]), i32([0] * 4), i32([3, 0, 0, 1]), i32([5, 6, 7, 8])
    big = torch.randn(8192, 8192, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    stream = torch.cuda.default_stream() if own else torch.cuda.Stream()
    assert (stream.cuda_stream == 0) == own
    with torch.cuda.stream(stream):
        for _ in range(20):
            big = (big @ big).clamp(-1, 1)
        parents.copy_(want)
        tokens.copy_(ids)
        bt.fork(parents, tokens, stream=stream.cuda_stream)
        parents.zero_()
        tokens.zero_()
    torch.cuda.synchronize()
    after = bt.tensor(name, np.float32).reshape(4, -1)
    for j, p in enumerate([3, 0, 0, 1]):
        np.testing.assert_array_equal(after[j], before[p])
    assert bt.tensor("token", np.int32).tolist() == [5, 6, 7, 8]
    bt.close()
    m.close()


def test_forks_captured_and_replayed():
    """A captured fork and its tokens, replayed with other parents, between the program's own eager steps of the device."""
    d = q35.make_dims(hidden=512, ffn=1536, vocab=8192, n_layers=4, lin_heads=4, attn_heads=4, kv_heads=2)
    m = q35.TextForCausalLM(d, seed=4, tmax=40)
    rng = np.random.default_rng(2)
    bt = q35.BatchDecoder(m, 4, 30)
    bt.generate([rng.integers(0, d.vocab, 7).astype(np.int32) for _ in range(4)], 0, prefill=True)
    names = ["layers.0.linear_attn.recurrent_state", "layers.0.linear_attn.conv_state", "layers.3.self_attn.k_cache", "hist"]
    read = lambda: [bt.tensor(n, np.int32).reshape(4, -1) for n in names]
    parents, tokens, status = i32([0, 1, 2, 3]), i32([0] * 4), torch.zeros(1, dtype=torch.int32, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        bt.fork(parents, tokens, status, torch.cuda.current_stream().cuda_stream)
    for p, t in (([3, 0, 0, 1], [5, 6, 7, 8]), ([1, -1, 3, 2], [9, -1, 8191, 0]), ([2, 2, 2, 2], [1, 2, 3, 4])):
        torch.cuda.synchronize()
        before = read()
        parents.copy_(i32(p))
        tokens.copy_(i32(t))
        graph.replay()
        torch.cuda.synchronize()
        after = read()
        for a, b, name in zip(after, before, names):
            want = b[[q if q >= 0 else j for j, q in enumerate(p)]]
            if name == "hist":
                want[:, 6] = np.maximum(t, 0)
            np.testing.assert_array_equal(a, want, name)
        assert bt.tensor("token", np.int32).tolist() == [max(x, 0) for x in t] and int(status) == 0
    bt.check()
    bt.close()
    m.close()

"""What BatchDecoder.fork does on the host: its waits and refusals (no GPU: the tensors and the library are stand-ins that
write down what is asked of them)."""
import types

import pytest
import torch

import q35
from q35 import _lib as L


class Rows:
    """As much of an int32 tensor of n rows on the GPU as a fork looks at."""
    is_cuda = True

    def __init__(self, n, dtype=torch.int32, is_cuda=True):
        self.shape, self.dtype, self.is_cuda = torch.Size([n]), dtype, is_cuda

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20


@pytest.fixture
def calls(monkeypatch):
    log = []
    lib = types.SimpleNamespace(q35_batch_fork=lambda h, p, st, stream: log.append(("fork", stream)) or 0,
                                q35_batch_set_tokens=lambda h, t, st, stream: log.append(("tokens", stream)) or 0)
    monkeypatch.setattr(L, "lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: log.append("stream")))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: log.append("device"))
    return log


@pytest.fixture
def batch():
    b = q35.BatchDecoder.__new__(q35.BatchDecoder)
    b.B, b.h = 3, None
    return b


@pytest.mark.parametrize("stream", [None, 0])
def test_forks_on_the_batchs_own_stream_wait(calls, batch, stream):
    """0 is the handle of torch's default stream; a null handle is the batch's own stream, which is not ordered with it."""
    batch.fork(Rows(3), Rows(3), stream=stream)
    assert [c if isinstance(c, str) else c[0] for c in calls] == ["stream", "fork", "tokens", "device"]


def test_forks_on_a_stream_do_not_wait(calls, batch):
    batch.fork(Rows(3), Rows(3), stream=4096)
    assert calls == [("fork", 4096), ("tokens", 4096)]


def test_check_of_no_batch():
    assert L.lib().q35_batch_check(None, None) == L.Q35_E_ARG and b"batch_check" in L.lib().q35_last_error()


@pytest.mark.parametrize("status", [Rows(1, torch.int64), Rows(1, torch.float32), Rows(1, is_cuda=False), Rows(0)])
def test_status_words_that_a_kernel_must_not_write_are_refused(calls, batch, status):
    with pytest.raises(AssertionError):
        batch.fork(Rows(3), Rows(3), status)
    assert calls == []
    batch.fork(Rows(3), Rows(3), Rows(1))
    assert len(calls) == 4

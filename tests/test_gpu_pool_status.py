"""A pool's status word under several streams."""
import threading
import time

import pytest
import torch

import q35

pytestmark = pytest.mark.gpu

L = q35._lib


def test_bits_of_another_stream_survive_a_check():
    """A check waits for its stream, which stays busy between its read of the word and the clearing; what a call on
    another stream reports in that time is left for the next check."""
    pool = q35.PagePool.empty(1, 2, kv_heads=1, page=16)
    a, b = (torch.zeros(1 << 28, device="cuda") for _ in range(2))  # 1 GiB
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()

    def copies(n):
        with torch.cuda.stream(busy):
            for _ in range(n):
                a.copy_(b)

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    args = i32(-1, -1, -1, -1)[None], i32(0), i32(-1), i32(48)

    def fork():  # three pages from a pool of two
        with torch.cuda.stream(other):
            return q35.pages_fork(pool, *args)

    torch.cuda.synchronize()
    fork()  # (its outputs' memory is there from here on)
    copies(2)
    busy.synchronize()
    t = time.perf_counter()
    copies(20)
    busy.synchronize()
    half = max(1, int(0.5 / ((time.perf_counter() - t) / 20)))  # copies of half a second
    pool.status.fill_(L.Q35_STATUS_ARG)
    torch.cuda.synchronize()
    told = []

    def check():
        with torch.cuda.stream(busy):
            try:
                pool.check()
            except q35.Q35Error as e:
                told.append(str(e))

    copies(half)
    read = torch.cuda.Event()
    read.record(busy)
    thread = threading.Thread(target=check)
    thread.start()
    time.sleep(0.2)
    copies(half)
    read.synchronize()
    time.sleep(0.1)
    f = fork()
    other.synchronize()
    assert not busy.query()  # (the clearing is still to come)
    thread.join()
    assert f.table.tolist() == [[0, 1, -1, -1]]
    assert len(told) == 1 and "Q35_E_RANGE" in told[0]
    with pytest.raises(q35.Q35Error, match="Q35_E_NOMEM"):
        pool.check()
    pool.check()


def test_check_takes_all_that_it_read():
    pool = q35.PagePool.empty(1, 2, kv_heads=1, page=16)
    for bits, error in ((L.Q35_STATUS_ARG, "Q35_E_RANGE"), (L.Q35_STATUS_FULL, "Q35_E_NOMEM"), (L.Q35_STATUS_ARG | L.Q35_STATUS_FULL, "Q35_E_RANGE")):
        pool.status.fill_(bits)
        with pytest.raises(q35.Q35Error, match=error):
            pool.check()
        pool.check()
        assert int(pool.status) == 0

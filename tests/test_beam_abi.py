"""Argument checks of the beams' entry points (before any GPU work: the pointers are numbers that nothing reads), and the
plain form of the selection on cases that can be told by hand."""
import ctypes

import numpy as np
import pytest
import torch

import beam_ref as B
import q35
from q35 import _lib as L

A = 1 << 20


def select(**kw):
    f = dict(x=1 << 30, dtype=L.Q35_F32, R=2, W=3, V=100, ld=100, scores=A, ended=None, k=4, so=A + 4096, parents=A + 8192, tokens=A + 12288,
             status=None, ws=A + 65536, nb=1 << 40, stream=None)
    f.update(kw)
    return L.lib().q35_beam_select(*f.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=L.Q35_Q4), L.Q35_E_ARG), (dict(dtype=3), L.Q35_E_ARG), (dict(R=0), L.Q35_E_SHAPE), (dict(W=0), L.Q35_E_SHAPE), (dict(W=257), L.Q35_E_SHAPE),
    (dict(V=0), L.Q35_E_SHAPE), (dict(V=(1 << 30) + 1, ld=1 << 31), L.Q35_E_SHAPE), (dict(ld=99), L.Q35_E_SHAPE), (dict(k=0), L.Q35_E_SHAPE),
    (dict(k=65), L.Q35_E_SHAPE), (dict(R=1 << 23), L.Q35_E_SHAPE),
    (dict(x=(1 << 30) + 2), L.Q35_E_ALIGN), (dict(x=(1 << 30) + 1, dtype=L.Q35_BF16), L.Q35_E_ALIGN), (dict(ws=None), L.Q35_E_WS),
    (dict(nb=100), L.Q35_E_WS), (dict(ws=A + 65537), L.Q35_E_ALIGN), (dict(so=A), L.Q35_E_ARG), (dict(so=A + 20), L.Q35_E_ARG), (dict(tokens=A + 8192 + 28), L.Q35_E_ARG),
    (dict(parents=(1 << 30) + 96), L.Q35_E_ARG), (dict(ended=A + 12288), L.Q35_E_ARG),
] + [(dict([(n, None)]), L.Q35_E_ARG) for n in ("x", "scores", "so", "parents", "tokens")])
def test_select_refusals(change, code):
    assert select(**change) == code
    assert b"beam_select" in L.lib().q35_last_error()


def test_select_ws_bytes():
    ws = L.lib().q35_beam_select_ws_bytes
    assert ws(1, 4, 248320, 8) > 0 and ws(1, 256, 1 << 23, 64) > 0
    for bad in ((0, 4, 100, 4), (1, 0, 100, 4), (1, 4, 0, 4), (1, 4, 100, 0), (1, 4, 100, 65), (1, 257, 100, 4), (1 << 16, 256, 100, 4)):
        assert ws(*bad) == 0


def fork(states=((A, A, 64, 64, 64),), parent=A, B=4, B_out=3, n=None):
    s = (L.State * max(1, len(states)))(*[L.State(*x) for x in states])
    return L.lib().q35_states_fork(s, len(states) if n is None else n, parent, B, B_out, None, None)


def test_states_refusals():
    far = A + (1 << 20)
    assert fork(()) == L.Q35_OK and fork(B_out=0) == L.Q35_OK
    assert fork(parent=None) == L.Q35_E_ARG
    assert fork(B=0) == L.Q35_E_SHAPE and fork(B=4097) == L.Q35_E_SHAPE and fork(B_out=-1) == L.Q35_E_SHAPE and fork(B_out=4097) == L.Q35_E_SHAPE
    assert fork(n=-1) == L.Q35_E_SHAPE
    assert fork(((None, A, 64, 64, 64),)) == L.Q35_E_ARG and fork(((A, None, 64, 64, 64),)) == L.Q35_E_ARG
    assert fork(((A, A, 32, 32, 64),)) == L.Q35_E_SHAPE and fork(((A, far, 64, 63, 64),)) == L.Q35_E_SHAPE and fork(((A, A, 64, 64, -1),)) == L.Q35_E_SHAPE
    assert fork(((A, A, 64, 128, 64),)) == L.Q35_E_ARG                      # in place with two strides
    assert fork(((A, A, 64, 64, 64), (A, far, 64, 64, 64))) == L.Q35_E_ARG  # one in place, one not
    assert fork(((A, A + 64, 64, 64, 64),)) == L.Q35_E_ARG                  # shifted by a row
    assert fork(((A, A + 255, 64, 64, 64),)) == L.Q35_E_ARG
    assert fork(((A, A, 64, 64, 64), (far, far, 64, 64, 64), (A, A, 64, 64, 64))) == L.Q35_E_ARG  # one twice
    assert L.lib().q35_states_fork(None, 1, A, 4, 3, None, None) == L.Q35_E_ARG


def test_selection_by_hand():
    # beam 0: probabilities 1/2, 1/4, 1/4; beam 1: 3/4, 1/4, 0
    with np.errstate(divide="ignore"):
        x = np.log(np.array([[2, 1, 1], [3, 1, 0]], np.float64)) + 7.0
    (s, p, t), _ = B.select(x, np.array([[0.0, np.log(0.5)]], np.float32), 6)
    np.testing.assert_allclose(np.exp(s[0, :5]), [0.5, 0.375, 0.25, 0.25, 0.125], rtol=1e-6)
    assert p[0].tolist() == [0, 1, 0, 0, 1, -1] and t[0].tolist() == [0, 0, 1, 2, 1, -1] and s[0, 5] == -np.inf
    (s, p, t), _ = B.select(x, np.array([[-np.inf, -1.0]], np.float32), 2, np.array([-1, 2]))
    assert p[0].tolist() == [1, -1] and t[0].tolist() == [2, -1] and s[0, 0] == -1.0
    B.check((s.astype(np.float32), p, t), x, np.array([[-np.inf, -1.0]], np.float32), 2, np.array([-1, 2]))
    with pytest.raises(AssertionError):
        B.check((s.astype(np.float32) + 1e-4, p, t), x, np.array([[-np.inf, -1.0]], np.float32), 2, np.array([-1, 2]))


def test_batch_forks_refuse_null_pointers():
    lib = L.lib()
    assert lib.q35_batch_fork(None, A, None, None) == L.Q35_E_ARG and lib.q35_batch_set_tokens(None, A, None, None) == L.Q35_E_ARG


def test_states_of_no_rows():
    none, two = torch.zeros(0, 8), torch.zeros(2, 8)
    parents = torch.zeros(0, dtype=torch.int32)
    assert q35.states_fork([none], parents)[0] is none
    assert q35.states_fork([none], parents, out=[two])[0] is two
    with pytest.raises(AssertionError):
        q35.states_fork([none], torch.full((2,), -1, dtype=torch.int32), out=[two])


def test_states_given_as_their_own_outputs_have_the_rows():
    """(More rows out than the tensors have would be written behind them.)"""
    s = torch.zeros(3, 8)
    with pytest.raises(AssertionError, match="3, 8"):
        q35.states_fork([s], torch.zeros(4, dtype=torch.int32), out=[s])

"""Argument checks of the paged caches' and the token scores' entry points: they refuse before any GPU work,
so the pointers here are numbers that nothing reads.  And the plain forms of tests/paged_ref.py on cases
that can be told by hand."""
import ctypes

import numpy as np
import pytest
import torch

import paged_ref as R
import q35
from q35 import _lib as L

A = 1 << 20  # a 16-byte aligned address


def pages(**kw):
    f = dict(data=A, dtype=L.Q35_BF16, n_layers=2, n_pages=100, kv_heads=2, page=64, head_dim=256)
    f.update(kw)
    return L.Pages(*[f[n] for n, _ in L.Pages._fields_])


BAD_POOLS = [(dict(data=None), L.Q35_E_ARG), (dict(dtype=3), L.Q35_E_ARG), (dict(dtype=-1), L.Q35_E_ARG), (dict(head_dim=128), L.Q35_E_SHAPE),
             (dict(page=8), L.Q35_E_SHAPE), (dict(page=48), L.Q35_E_SHAPE), (dict(page=512), L.Q35_E_SHAPE), (dict(page=0), L.Q35_E_SHAPE),
             (dict(n_layers=0), L.Q35_E_SHAPE), (dict(n_pages=0), L.Q35_E_SHAPE), (dict(n_pages=262145), L.Q35_E_SHAPE),
             (dict(kv_heads=0), L.Q35_E_SHAPE), (dict(data=A + 8), L.Q35_E_ALIGN)]


def attention(**kw):
    d = q35.make_dims(**{k: kw.pop(k) for k in ("attn_heads", "kv_heads", "head_dim", "rot_dim") if k in kw})
    f = dict(pool=pages(), layer=1, qg=A, ld_qg=4096, k=A, v=A, kv_ld=512, T=3, start=A, pos=A, B=2, table=A, ld_table=5, qw=A, kw=A, cos=A, sin=A,
             rows=300, out=A, ld_out=2048, status=None, ws=A, ws_bytes=1 << 40, stream=None)
    f.update(kw)
    return L.lib().q35_attention_core_paged(ctypes.byref(d), *f.values())


@pytest.mark.parametrize("change,code", [
    (dict(layer=2), L.Q35_E_SHAPE), (dict(layer=-1), L.Q35_E_SHAPE), (dict(T=0), L.Q35_E_SHAPE), (dict(B=0), L.Q35_E_SHAPE), (dict(T=-4), L.Q35_E_SHAPE),
    (dict(T=(1 << 20) + 1), L.Q35_E_SHAPE), (dict(ld_table=0), L.Q35_E_SHAPE), (dict(rows=0), L.Q35_E_SHAPE), (dict(ld_qg=4092), L.Q35_E_SHAPE),
    (dict(kv_ld=508), L.Q35_E_SHAPE), (dict(ld_out=2044), L.Q35_E_SHAPE), (dict(ld_qg=4097), L.Q35_E_ALIGN), (dict(kv_ld=514), L.Q35_E_ALIGN),
    (dict(ld_out=2049), L.Q35_E_ALIGN), (dict(qg=A + 4), L.Q35_E_ALIGN), (dict(k=A + 4), L.Q35_E_ALIGN), (dict(out=A + 8), L.Q35_E_ALIGN),
    (dict(qw=A + 4), L.Q35_E_ALIGN), (dict(ws=None), L.Q35_E_WS), (dict(ws_bytes=0), L.Q35_E_WS), (dict(ws=A + 4), L.Q35_E_ALIGN),
    (dict(kv_heads=4), L.Q35_E_SHAPE), (dict(attn_heads=7), L.Q35_E_SHAPE), (dict(attn_heads=34), L.Q35_E_SHAPE), (dict(rot_dim=63), L.Q35_E_SHAPE),
    (dict(rot_dim=258), L.Q35_E_SHAPE), (dict(rot_dim=0), L.Q35_E_SHAPE), (dict(head_dim=128), L.Q35_E_SHAPE),
] + [(dict([(n, None)]), L.Q35_E_ARG) for n in ("qg", "k", "v", "start", "pos", "table", "qw", "kw", "cos", "sin", "out")])
def test_attention_refusals(change, code):
    assert attention(**change) == code
    assert b"attention_paged" in L.lib().q35_last_error()


@pytest.mark.parametrize("change,code", BAD_POOLS)
def test_bad_pools(change, code):
    assert attention(pool=pages(**change)) == code
    assert L.lib().q35_pages_copy(pages(), pages(**change), A, A, 1, None, A, 64, None) in (code, L.Q35_E_SHAPE)
    assert L.lib().q35_pages_copy(pages(**change), pages(), A, A, 1, None, A, 64, None) in (code, L.Q35_E_SHAPE)
    assert fork(pool=pages(**change)) == code
    assert compact(pool=pages(**change)) == code


def test_copy_refusals():
    lib = L.lib()

    def copy(src=pages(), dst=pages(), s=A, d=A, n=3, ws=A, nb=64):
        return lib.q35_pages_copy(src, dst, s, d, n, None, ws, nb, None)

    size = 2 * 100 * 2 * 2 * 64 * 256 * 2
    assert copy(n=0) == L.Q35_OK
    assert copy(n=-1) == L.Q35_E_SHAPE
    assert copy(s=None) == L.Q35_E_ARG and copy(d=None) == L.Q35_E_ARG
    assert copy(n=257, ws=None, nb=300) == L.Q35_E_WS and copy(n=257, nb=256) == L.Q35_E_WS
    assert copy(n=1 << 30, nb=1 << 40) == L.Q35_E_SHAPE
    for other in (dict(dtype=L.Q35_F16), dict(n_layers=1), dict(kv_heads=1), dict(page=32)):
        assert copy(dst=pages(data=A + 4 * size, **other)) == L.Q35_E_SHAPE
    assert copy(dst=pages(n_pages=90)) == L.Q35_E_ARG
    assert copy(dst=pages(data=A + size - 16)) == L.Q35_E_ARG
    assert copy(dst=pages(data=A + 16)) == L.Q35_E_ARG


def fork(**kw):
    f = dict(pool=pages(), table=A, ld=4, len=A, B=3, parent=A, grow=None, B_out=5, out=A + 4096, len_out=A + 8192, refs=A, status=None, stream=None)
    f.update(kw)
    return L.lib().q35_pages_fork(*f.values())


@pytest.mark.parametrize("change,code", [
    (dict(B=0), L.Q35_E_SHAPE), (dict(B=4097), L.Q35_E_SHAPE), (dict(B_out=0), L.Q35_E_SHAPE), (dict(B_out=4097), L.Q35_E_SHAPE), (dict(ld=0), L.Q35_E_SHAPE),
    (dict(ld=65537), L.Q35_E_SHAPE), (dict(out=A), L.Q35_E_ARG), (dict(out=A + 44), L.Q35_E_ARG), (dict(out=A - 40), L.Q35_E_ARG), (dict(len_out=A), L.Q35_E_ARG),
] + [(dict([(n, None)]), L.Q35_E_ARG) for n in ("table", "len", "parent", "out", "len_out", "refs")])
def test_fork_refusals(change, code):
    assert fork(**change) == code


def compact(**kw):
    f = dict(pool=pages(), table=A, ld=4, B=3, out=A + 4096, refs=A, used=A, status=None, ws=A, nb=804, stream=None)
    f.update(kw)
    return L.lib().q35_pages_compact(*f.values())


@pytest.mark.parametrize("change,code", [
    (dict(B=0), L.Q35_E_SHAPE), (dict(ld=0), L.Q35_E_SHAPE), (dict(ld=65537), L.Q35_E_SHAPE), (dict(out=A), L.Q35_E_ARG), (dict(out=A + 44), L.Q35_E_ARG),
    (dict(ws=None), L.Q35_E_WS), (dict(nb=803), L.Q35_E_WS), (dict(ws=A + 2), L.Q35_E_ALIGN),
] + [(dict([(n, None)]), L.Q35_E_ARG) for n in ("table", "out", "refs", "used")])
def test_compact_refusals(change, code):
    assert compact(**change) == code


def score(**kw):
    f = dict(x=A, dtype=L.Q35_F32, M=2, V=100, ld=100, targets=None, top=3, logprob=None, rank=None, entropy=A, ids=A, lps=A, status=None, ws=A, nb=1 << 40,
             stream=None)
    f.update(kw)
    return L.lib().q35_token_logprobs(*f.values())


@pytest.mark.parametrize("change,code", [
    (dict(x=None), L.Q35_E_ARG), (dict(entropy=None), L.Q35_E_ARG), (dict(dtype=5), L.Q35_E_ARG), (dict(M=0), L.Q35_E_SHAPE), (dict(V=0), L.Q35_E_SHAPE),
    (dict(ld=99), L.Q35_E_SHAPE), (dict(top=-1), L.Q35_E_SHAPE), (dict(top=65), L.Q35_E_SHAPE), (dict(V=2, top=3), L.Q35_E_SHAPE), (dict(ids=None), L.Q35_E_ARG),
    (dict(lps=None), L.Q35_E_ARG), (dict(targets=A), L.Q35_E_ARG), (dict(targets=A, rank=A), L.Q35_E_ARG), (dict(targets=A, logprob=A), L.Q35_E_ARG),
    (dict(x=A + 2), L.Q35_E_ALIGN), (dict(dtype=L.Q35_F16, x=A + 1), L.Q35_E_ALIGN), (dict(ws=None), L.Q35_E_WS), (dict(nb=16), L.Q35_E_WS),
    (dict(ws=A + 8), L.Q35_E_ALIGN), (dict(V=(1 << 30) + 1, ld=1 << 31), L.Q35_E_SHAPE),
])
def test_score_refusals(change, code):
    assert score(**change) == code


def test_status_check_refuses_null():
    assert L.lib().q35_status_check(None, None) == L.Q35_E_ARG


def test_workspace_sizes():
    d = q35.dims_2b()
    lib = L.lib()
    assert lib.q35_attention_paged_ws_bytes(ctypes.byref(d), 0, 1) == 0 and lib.q35_attention_paged_ws_bytes(None, 1, 1) == 0
    assert lib.q35_attention_paged_ws_bytes(ctypes.byref(d), 1, 1) > 0
    assert lib.q35_pages_copy_ws_bytes(0) == 0 and lib.q35_pages_copy_ws_bytes(700) >= 700
    assert lib.q35_pages_compact_ws_bytes(0) == 0 and lib.q35_pages_compact_ws_bytes(100) >= 804
    assert lib.q35_token_logprobs_ws_bytes(0, 5, 1) == 0 and lib.q35_token_logprobs_ws_bytes(1, 248320, 64) > 0


def test_python_surface_refuses_host_tensors_and_wrong_shapes():
    with pytest.raises(AssertionError):
        q35.PagePool(torch.zeros(1, 4, 2, 1, 16, 256))
    with pytest.raises(AssertionError):
        q35.PagePool(torch.zeros(4, 2, 1, 16, 256))
    with pytest.raises(AssertionError):
        q35.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(AssertionError):
        q35.token_logprobs(torch.zeros(2, 10, dtype=torch.float64))


def test_plain_forms_by_hand():
    rows, lens, refs, copies, short = R.fork([[4, 2, -1], [7, -1, -1]], [20, 16], [0, 0, 1, -1], [0, 1, 20, 1], 9, 16)
    # row 0 keeps the half-full page 2, row 1 gets page 0 as its copy; row 2 two new ones; row 3 starts with one
    assert rows == [[4, 2, -1], [4, 0, -1], [7, 1, 3], [5, -1, -1]] and lens == [20, 20, 16, 0]
    assert copies == [(2, 0, 4)] and not short and refs == [1, 1, 1, 1, 2, 1, 0, 1, 0]
    assert R.compact([[5, 1], [5, -1], [7, 0]], 8) == ([[2, 1], [2, -1], [3, 0]], [1, 1, 2, 1, 0, 0, 0, 0], 4, [(5, 2), (7, 3)])
    lp, rank, ent, ids, tlp = R.scores(np.log(np.array([[0.5, 0.25, 0.25]])), [2], 2)
    np.testing.assert_allclose([lp[0], ent[0], *tlp[0]], [np.log(0.25), 1.5 * np.log(2), np.log(0.5), np.log(0.25)], rtol=1e-12)
    assert rank[0] == 2 and ids[0].tolist() == [0, 1]


def test_plain_attention_against_an_independent_one():
    """The oracle's own checks: one key gives its value, equal keys their mean, the gate halves at 0."""
    d = q35.make_dims(attn_heads=2, kv_heads=1, rot_dim=64)
    r = np.random.default_rng(0)
    pool = torch.zeros(1, 3, 2, 1, 16, 256)
    k = np.repeat(r.standard_normal((1, 256)), 3, 0).astype(np.float32)
    v = r.standard_normal((3, 256)).astype(np.float32)
    qg = np.concatenate([r.standard_normal((3, 256)), np.zeros((3, 256))] * 2, 1).astype(np.float32)
    one, zero = np.ones((3, 64), np.float32), np.zeros((3, 64), np.float32)
    w = np.zeros(256, np.float32)
    out, tol = R.attention(d, pool, 0, qg, k, v, [0, 3], [0], [[2]], w, w, one, zero)
    want = np.cumsum(v, 0) / np.arange(1, 4)[:, None] / 2
    np.testing.assert_allclose(out, np.concatenate([want, want], 1), atol=1e-6)
    assert torch.equal(pool[0, 2, 1, 0, :3], torch.from_numpy(v)) and (pool[0, :2] == 0).all() and tol.min() > 0


def test_limits():
    """Heads, rotary rows, table entries and launch sizes beyond what the kernels index."""
    assert attention(attn_heads=2048, kv_heads=128, pool=pages(kv_heads=128), ld_qg=1 << 20, kv_ld=1 << 15, ld_out=1 << 19) == L.Q35_E_SHAPE
    assert attention(rows=(1 << 30) + 1) == L.Q35_E_SHAPE
    wide = dict(attn_heads=64, kv_heads=16)
    big = dict(wide, pool=pages(kv_heads=16), T=1 << 20, ld_qg=1 << 15, kv_ld=1 << 12, ld_out=1 << 14)  # T (heads + kv heads) > 2^25
    assert attention(**big) == L.Q35_E_SHAPE
    ws = L.lib().q35_attention_paged_ws_bytes
    assert ws(ctypes.byref(q35.make_dims(**wide)), 1 << 20, 4) == 0
    for bad in (dict(kv_heads=0), dict(attn_heads=0), dict(attn_heads=1, kv_heads=2), dict(attn_heads=-8), dict(attn_heads=2048, kv_heads=128), dict(attn_heads=34)):
        assert ws(ctypes.byref(q35.make_dims(**bad)), 4, 4) == 0, bad
    assert ws(ctypes.byref(q35.dims_2b()), (1 << 20) + 1, 4) == 0 and ws(ctypes.byref(q35.dims_2b()), 4, (1 << 20) + 1) == 0
    assert fork(ld=65536, B=1, B_out=1025, out=A + (1 << 28)) == L.Q35_E_SHAPE
    assert fork(len_out=A + 8) == L.Q35_E_ARG  # the last of len's three
    assert fork(parent=A + 8192) == L.Q35_E_ARG and fork(grow=A + 8192 + 16) == L.Q35_E_ARG  # len_out's place
    assert compact(ld=65536, B=1025, out=A + (1 << 30)) == L.Q35_E_SHAPE
    one = pages(n_layers=1, kv_heads=1, page=256, dtype=L.Q35_F32)  # 32 units of 16 KB per page
    assert L.lib().q35_pages_copy(one, one, A, A, 1 << 19, None, A, 1 << 40, None) == L.Q35_E_SHAPE
    assert score(M=1 << 24, top=0) == L.Q35_E_SHAPE

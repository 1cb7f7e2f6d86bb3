"""Argument checks of the 4-bit caches' entry points (before any GPU work) and the plain form of their rows on cases that can
be told by hand."""
import ctypes

import numpy as np
import pytest

import q35
import q4_ref as Q
from q35 import _lib as L

A = 1 << 20


def pages(**kw):
    f = dict(data=A, dtype=L.Q35_Q4, n_layers=2, n_pages=100, kv_heads=2, page=64, head_dim=256)
    f.update(kw)
    return L.Pages(*[f[n] for n, _ in L.Pages._fields_])


def read(**kw):
    f = dict(pool=pages(), layer=1, table=A, ld=5, B=2, row=A, pos=A, n=3, out=A, status=None, stream=None)
    f.update(kw)
    return L.lib().q35_pages_read(*f.values())


@pytest.mark.parametrize("change,code", [
    (dict(layer=2), L.Q35_E_SHAPE), (dict(layer=-1), L.Q35_E_SHAPE), (dict(n=-1), L.Q35_E_SHAPE), (dict(B=0), L.Q35_E_SHAPE), (dict(ld=0), L.Q35_E_SHAPE),
    (dict(n=1 << 24), L.Q35_E_SHAPE), (dict(out=A + 8), L.Q35_E_ALIGN), (dict(pool=pages(dtype=3)), L.Q35_E_ARG), (dict(pool=pages(dtype=5)), L.Q35_E_ARG),
    (dict(pool=pages(head_dim=144)), L.Q35_E_SHAPE), (dict(pool=pages(data=A + 8)), L.Q35_E_ALIGN), (dict(pool=pages(page=24)), L.Q35_E_SHAPE),
] + [(dict([(n, None)]), L.Q35_E_ARG) for n in ("table", "row", "pos", "out")])
def test_read_refusals(change, code):
    assert read(**change) == code
    assert b"pages_read" in L.lib().q35_last_error()


def test_read_of_nothing():
    assert read(n=0, row=None, pos=None, out=None) == L.Q35_OK


def test_copies_between_types_and_overlapping_pools_are_refused():
    copy = lambda src, dst, n=3: L.lib().q35_pages_copy(src, dst, A, A, n, None, A, 64, None)
    size = 2 * 100 * 2 * 2 * 64 * 144
    assert copy(pages(), pages(data=A + 4 * size, dtype=L.Q35_F16)) == L.Q35_E_SHAPE
    assert copy(pages(), pages(data=A + size - 16)) == L.Q35_E_ARG
    assert copy(pages(), pages(data=A + size), 1 << 30) == L.Q35_E_SHAPE  # (beside each other: the count is what is refused)


def test_attention_refuses_other_shapes():
    d = q35.make_dims(kv_heads=4)
    f = [ctypes.byref(d), pages(), 1, A, 4096, A, A, 512, 3, A, A, 2, A, 5, A, A, A, A, 300, A, 2048, None, A, 1 << 40, None]
    assert L.lib().q35_attention_core_paged(*f) == L.Q35_E_SHAPE


def test_rows_by_hand():
    v = np.zeros(256, np.float32)
    v[:32] = np.minimum(np.arange(32), 15)          # scale 1, zero 0
    v[32:64] = np.clip(np.arange(32) / 2 - 7.5, -7.5, 7.5)  # scale 1, zero 8 (7.5 to even), codes rounded to even
    v[64:96] = -30.0                                # scale 2, zero 15
    v[96] = 15.1                                    # 15.1 / 15 = 1.00667: 1 + 1/64
    v[128] = np.inf
    v[160] = 15 * 2.0 ** -21                        # below the smallest scale, 2^-20
    row = Q.pack(v)
    assert row[:16].tolist() == [0x10, 0x32, 0x54, 0x76, 0x98, 0xBA, 0xDC, 0xFE] + [0xFF] * 8
    words = row[128:].view(np.uint16).tolist()
    assert words == [0x3C00, 0x3C08, 0x400F, 0x3C10, 0x7FF0, 0x0010, 0, 0]
    w = Q.unpack(row)
    assert w[:32].tolist() == v[:32].tolist() and w[64:96].tolist() == [-30.0] * 32 and np.isnan(w[128:160]).all()
    assert w[32:36].tolist() == [-8.0, -7.0, -6.0, -6.0] and w[63] == 7.0  # -7.5, -7, -6.5, -6; 7.5 cut at 15 - 8
    assert w[96] == 15 * (1 + 1 / 64) and w[160] == 8 * 2.0 ** -20  # (7.5 to even)
    assert np.array_equal(Q.unpack(row).astype(np.float16).astype(np.float64), w, equal_nan=True)
    # packing what a row stands for gives the same values again
    x = np.random.default_rng(0).standard_normal((40, 256)).astype(np.float32)
    once = Q.unpack(Q.pack(x))
    assert np.abs(once - x).max() < 0.25

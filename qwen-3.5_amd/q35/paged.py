"""Caches in pages, and scores of tokens: what a program needs that serves several continuations of shared
contexts (beam search, several samples of a prompt, drafted tokens, prompt chunks beside decoding
sequences).  No counterparts in the reference, which decodes one sequence greedily.

  attention_core_paged  attention_core_prefill / _decode for any mix of sequences over a PagePool
  pages_fork            the next page table: forked, dropped, freed and reserved sequences
  pages_copy            pages copied within a pool or between two
  pages_compact         the pages in use moved to the pool's front
  token_logprobs        log probabilities, ranks, entropy and the highest alternatives of logits

    pool = q35.PagePool.empty(6, 4096)
    f = q35.pages_fork(pool, table, lens, parents, grow)       # f.table, f.lens, f.refs
    out = q35.attention_core_paged(dims, pool, layer, q_gate, k_new, v_new, start, f.lens, f.table, ...)
    pool.check()                                               # optional: raises what the kernels refused

All calls are asynchronous on the current stream of their tensors' device; their scratch comes from
torch's allocator call by call, so calls on several streams and captured graphs share nothing but what they are
given: the pool's pages, and its status word, to which calls only add and from which a check takes what it read.
"""
import collections
import contextlib
import ctypes
import functools

import torch

from . import _lib as L
from .kernels import _stream

_DTYPES = {torch.float32: L.Q35_F32, torch.float16: L.Q35_F16, torch.bfloat16: L.Q35_BF16}
_HERE = contextlib.nullcontext()

PagesFork = collections.namedtuple("PagesFork", "table lens refs")
PagesCompact = collections.namedtuple("PagesCompact", "table refs used")
TokenLogprobs = collections.namedtuple("TokenLogprobs", "logprob rank entropy top_ids top_logprobs")


def _on(first, *tensors):
    """The tensors' device as the current one (they must share it)."""
    dev = first.get_device()
    assert dev >= 0, "tensors must be on the GPU"
    for t in tensors:
        assert t is None or t.get_device() == dev, "tensors on different devices"
    return _HERE if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _ints(t, *shape):
    """An int32 tensor of the shape, contiguous."""
    assert t.dtype is torch.int32 and t.shape == shape, (t.dtype, tuple(t.shape), shape)
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


@functools.lru_cache(maxsize=1024)
def _score_ws_bytes(M, V, top):
    return L.lib().q35_token_logprobs_ws_bytes(M, V, top)


class PagePool:
    """Pages of the attention layers' caches: data [n_layers, n_pages, 2, kv_heads, page, 256] in float32,
    float16 or bfloat16 (plane 0 the keys after norm and rotary, plane 1 the values); page a power of
    two in 16..256.  Who owns which page is the page tables' matter (int32 [B, entries], -1 none)."""

    def __init__(self, data):
        assert data.dim() == 6 and data.shape[2] == 2 and data.is_contiguous() and data.dtype in _DTYPES, \
            (tuple(data.shape), data.dtype)
        assert data.device.type == "cuda", "the pool must be on the GPU"
        self.data = data
        self.n_layers, self.n_pages, _, self.kv_heads, self.page, self.head_dim = data.shape
        self.status = torch.zeros(1, dtype=torch.int32, device=data.device)
        self._desc = L.Pages(data.data_ptr(), _DTYPES[data.dtype], self.n_layers, self.n_pages, self.kv_heads, self.page,
                             self.head_dim)

    @classmethod
    def empty(cls, n_layers, n_pages, kv_heads=2, page=64, head_dim=256, dtype=torch.float32, device="cuda"):
        return cls(torch.empty((n_layers, n_pages, 2, kv_heads, page, head_dim), dtype=dtype, device=device))

    def desc(self):
        return self._desc

    def check(self):
        """Synchronise the current stream and raise Q35Error if a call on this pool met an index out of range
        (Q35_E_RANGE) or found no free page (Q35_E_NOMEM) since the last check."""
        with _on(self.data):
            L.check(L.lib().q35_status_check(self.status.data_ptr(), _stream()))


def attention_core_paged(dims, pool, layer, q_gate, k_new, v_new, seq_start, pos, table, q_norm, k_norm, rope_cos, rope_sin,
                         out=None, check=False):
    """q/k norm, RoPE, append to the pages, causal GQA attention and sigmoid gate for the new tokens of B
    sequences: rows seq_start[b] .. seq_start[b+1]-1 (int32 [B+1]) are sequence b's, at positions pos[b] ..
    (int32 [B]: tokens cached before); table int32 [B, entries].  q_gate [T, heads*512]; k_new / v_new
    [T, kv_heads*256]; rotary tables [rows, rot_dim]; returns [T, heads*256] (rows of no sequence are left
    as they are in `out`).  check=True synchronises and raises as PagePool.check does."""
    T, B = q_gate.shape[0], pos.shape[0]
    H, KV, hd, rot, f32 = dims.attn_heads, dims.kv_heads, dims.head_dim, dims.rot_dim, torch.float32
    assert q_gate.dtype is k_new.dtype is v_new.dtype is f32, (q_gate.dtype, k_new.dtype, v_new.dtype)
    assert q_gate.shape == (T, 2 * H * hd) and k_new.shape == (T, KV * hd) == v_new.shape, \
        (tuple(q_gate.shape), tuple(k_new.shape), tuple(v_new.shape))
    (ld_q, cq), (ld_k, ck), (ld_v, cv) = q_gate.stride(), k_new.stride(), v_new.stride()
    assert cq == ck == cv == 1, "rows must be contiguous"
    if T <= 1:  # (the stride of a single row says nothing)
        ld_q, ld_k, ld_v = 2 * H * hd, KV * hd, KV * hd
    assert ld_k == ld_v, "k_new and v_new must have one row stride"
    rows = rope_cos.shape[0]
    assert q_norm.shape == (hd,) == k_norm.shape and rope_cos.shape == (rows, rot) == rope_sin.shape
    for w in (q_norm, k_norm, rope_cos, rope_sin):
        assert w.dtype is f32 and w.is_contiguous(), (w.dtype, w.stride())
    if out is None:
        out = torch.empty(T, H * hd, dtype=f32, device=q_gate.device)
    assert out.dtype is f32 and out.shape == (T, H * hd) and out.stride(1) == 1, (tuple(out.shape), out.dtype, out.stride())
    width = table.shape[1]
    seq_start, pos, table = _ints(seq_start, B + 1), _ints(pos, B), _ints(table, B, width)
    if T == 0 or B == 0:
        return out
    lib, d = L.lib(), ctypes.byref(dims)
    with _on(q_gate, pool.data, k_new, v_new, seq_start, pos, table, q_norm, k_norm, rope_cos, rope_sin, out):
        nbytes = lib.q35_attention_paged_ws_bytes(d, T, B)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q_gate.device)
        L.check(lib.q35_attention_core_paged(
            d, pool.desc(), layer, q_gate.data_ptr(), ld_q, k_new.data_ptr(), v_new.data_ptr(), ld_k, T, seq_start.data_ptr(),
            pos.data_ptr(), B, table.data_ptr(), width, q_norm.data_ptr(), k_norm.data_ptr(), rope_cos.data_ptr(),
            rope_sin.data_ptr(), rows, out.data_ptr(), out.stride(0) if T > 1 else H * hd, pool.status.data_ptr(), ws.data_ptr(),
            nbytes, _stream()))
    if check:
        pool.check()
    return out


def pages_copy(pool, src, dst, to=None, check=False):
    """Copies page src[i] of `pool` to page dst[i] of `to` (default: the same pool) in every layer; src and
    dst int32 [n].  Pairs that name a page outside their pool, a destination twice or, in one pool, a page
    as source and destination are not copied (PagePool.check of the destination's pool raises)."""
    to = pool if to is None else to
    n = src.shape[0]
    src, dst = _ints(src, n), _ints(dst, n)
    with _on(pool.data, to.data, src, dst):
        # (up to 256 pairs need no scratch)
        ws = torch.empty(n, dtype=torch.uint8, device=src.device) if n > 256 else None
        L.check(L.lib().q35_pages_copy(pool.desc(), to.desc(), src.data_ptr(), dst.data_ptr(), n, to.status.data_ptr(),
                                       _ptr(ws), n, _stream()))
    if check:
        to.check()


def pages_fork(pool, table, lens, parents, grow=None, check=False):
    """The page table of the next set of sequences: row j continues sequence parents[j] of `table` (-1: an
    empty row) with pages for grow[j] more tokens.  Full pages are shared; a partly filled last page stays with the
    first row that continues it, unless a row names it as a full page, and every other row gets a copy.  table int32 [B, entries], lens int32 [B],
    parents and grow int32 [B_out].  Returns PagesFork(table [B_out, entries], lens [B_out], refs [n_pages]:
    the rows that name each page).  `table` must cover every sequence that is to live on; it stays as
    it was.  check=True raises Q35Error where no page was left (Q35_E_NOMEM) or an index was out of range."""
    B, n = table.shape
    Bo = parents.shape[0]
    table, lens, parents = _ints(table, B, n), _ints(lens, B), _ints(parents, Bo)
    if grow is not None:
        grow = _ints(grow, Bo)
    dev = table.device
    with _on(pool.data, table, lens, parents, grow):
        res = PagesFork(torch.empty(Bo, n, dtype=torch.int32, device=dev), torch.empty_like(parents),
                        torch.empty(pool.n_pages, dtype=torch.int32, device=dev))
        L.check(L.lib().q35_pages_fork(pool.desc(), table.data_ptr(), n, lens.data_ptr(), B, parents.data_ptr(),
                                       grow.data_ptr() if grow is not None else None, Bo, res.table.data_ptr(),
                                       res.lens.data_ptr(), res.refs.data_ptr(), pool.status.data_ptr(), _stream()))
    if check:
        pool.check()
    return res


def pages_compact(pool, table, check=False):
    """Moves the pages that `table` (int32 [B, entries]) names to the pool's front in every layer; returns
    PagesCompact(table, refs [n_pages], used int32 [1]: pages from there on are free)."""
    B, n = table.shape
    table = _ints(table, B, n)
    dev = table.device
    with _on(pool.data, table):
        res = PagesCompact(torch.empty_like(table), torch.empty(pool.n_pages, dtype=torch.int32, device=dev),
                           torch.empty(1, dtype=torch.int32, device=dev))
        nbytes = L.lib().q35_pages_compact_ws_bytes(pool.n_pages)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        L.check(L.lib().q35_pages_compact(pool.desc(), table.data_ptr(), n, B, res.table.data_ptr(), res.refs.data_ptr(),
                                          res.used.data_ptr(), pool.status.data_ptr(), ws.data_ptr(), nbytes, _stream()))
    if check:
        pool.check()
    return res


def token_logprobs(logits, targets=None, top=0, check=False):
    """Scores of logits [..., V] (float32, float16 or bfloat16): TokenLogprobs of logprob and rank [...] of
    targets (int32 [...]; None without; a negative target scores 0 with rank -1), entropy [...] in nats, and
    top_ids / top_logprobs [..., top], highest first and the lowest id first among equal logits.
    rank counts the tokens before the target in that order.  check=True synchronises and raises Q35Error
    (Q35_E_RANGE) for a target >= V, which otherwise scores NaN with rank -1."""
    V, lead = logits.shape[-1], logits.shape[:-1]
    dtype, dev, f32, i32 = _DTYPES.get(logits.dtype), logits.device, torch.float32, torch.int32
    assert dtype is not None, logits.dtype
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)  # (a view where the rows have one stride)
    if x.stride(1) != 1 or x.stride(0) < V:
        x = x.contiguous()
    M = x.shape[0]
    if targets is not None:
        targets = _ints(targets, *lead)
    with _on(x, targets):
        logprob = rank = ids = lps = status = None
        entropy = torch.empty(*lead, dtype=f32, device=dev) if lead else torch.empty((), dtype=f32, device=dev)
        if targets is not None:
            logprob, rank = torch.empty_like(entropy), torch.empty_like(targets)
        if top:
            ids = torch.empty(*lead, top, dtype=i32, device=dev)
            lps = torch.empty_like(ids, dtype=f32)
        res = TokenLogprobs(logprob, rank, entropy, ids, lps)
        if M == 0:
            return res
        if check:
            status = torch.zeros(1, dtype=i32, device=dev)
        nbytes = _score_ws_bytes(M, V, top)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        L.check(L.lib().q35_token_logprobs(x.data_ptr(), dtype, M, V, x.stride(0) if M > 1 else V, _ptr(targets), top, _ptr(logprob),
                                           _ptr(rank), entropy.data_ptr(), _ptr(ids), _ptr(lps), _ptr(status), ws.data_ptr(),
                                           nbytes, _stream()))
        if check:
            L.check(L.lib().q35_status_check(status.data_ptr(), _stream()))
    return res

"""Caches in pages, and scores of tokens: what a program needs that serves several continuations of shared
contexts (beam search, several samples of a prompt, drafted tokens, prompt chunks beside decoding
sequences).  No counterparts in the reference, which decodes one sequence greedily.

  attention_core_paged  attention_core_prefill / _decode for any mix of sequences over a PagePool
  pages_read            what a pool holds of given tokens, as values
  pages_fork            the next page table: forked, dropped, freed and reserved sequences
  pages_copy            pages copied within a pool or between two
  pages_compact         the pages in use moved to the pool's front
  states_fork           the same for states that are one row per sequence
  beam_select           the next beams: the highest continuations of each group of beams
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
import struct

import torch

from . import _lib as L
from .kernels import _stream

_DTYPES = {torch.float32: L.Q35_F32, torch.float16: L.Q35_F16, torch.bfloat16: L.Q35_BF16}
Q4 = "q4"       # the dtype of a pool in 4 bits
_Q4_ROW = 144   # bytes that it has for a token of a head: 256 codes, a 16-bit word for each 32
_HERE = contextlib.nullcontext()

PagesFork = collections.namedtuple("PagesFork", "table lens refs")
PagesCompact = collections.namedtuple("PagesCompact", "table refs used")
BeamSelect = collections.namedtuple("BeamSelect", "scores parents tokens")
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
def _attention_ws_bytes(heads, kv_heads, T, B, device):
    """(By device: it goes by the compute units of the current one.)"""
    return L.lib().q35_attention_paged_ws_bytes(ctypes.byref(L.make_dims(attn_heads=heads, kv_heads=kv_heads)), T, B)


@functools.lru_cache(maxsize=1024)
def _score_ws_bytes(M, V, top):
    return L.lib().q35_token_logprobs_ws_bytes(M, V, top)


@functools.lru_cache(maxsize=1024)
def _beam_ws_bytes(G, W, V, k):
    return L.lib().q35_beam_select_ws_bytes(G, W, V, k)


class PagePool:
    """Pages of the attention layers' caches: data [n_layers, n_pages, 2, kv_heads, page, 256] in float32,
    float16 or bfloat16 (plane 0 the keys after norm and rotary, plane 1 the values); page a power of
    two in 16..256.  Who owns which page is the page tables' matter (int32 [B, entries], -1 none).

    A pool in 4 bits (dtype=q35.Q4) has uint8 rows of 144 bytes instead of 256 values: 256 codes and a 16-bit word (a scale
    and a zero) for each 32 of them, as include/q35.h lays them out: 28% of a 16-bit pool's bytes, and each value off by
    about 1/30 of its 32 values' range at most.  pages_read gives rows as values."""

    def __init__(self, data):
        q4 = data.dtype is torch.uint8
        assert data.dim() == 6 and data.shape[2] == 2 and data.is_contiguous() and (data.dtype in _DTYPES or q4), \
            (tuple(data.shape), data.dtype)
        assert not q4 or data.shape[5] == _Q4_ROW, tuple(data.shape)
        assert data.device.type == "cuda", "the pool must be on the GPU"
        self.data = data
        self.n_layers, self.n_pages, _, self.kv_heads, self.page, self.head_dim = data.shape
        if q4:
            self.head_dim = 256
        self.status = torch.zeros(1, dtype=torch.int32, device=data.device)
        self._desc = L.Pages(data.data_ptr(), L.Q35_Q4 if q4 else _DTYPES[data.dtype], self.n_layers, self.n_pages, self.kv_heads,
                             self.page, self.head_dim)

    @classmethod
    def empty(cls, n_layers, n_pages, kv_heads=2, page=64, head_dim=256, dtype=torch.float32, device="cuda"):
        if dtype == Q4:
            assert head_dim == 256, head_dim
            head_dim, dtype = _Q4_ROW, torch.uint8
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
    as they are in `out`).  The kernels are chosen by what `table` and the rotary tables have room for: give those of the longest
    sequence, not of the longest possible, where that is known.  check=True synchronises and raises as PagePool.check does."""
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
        nbytes = _attention_ws_bytes(H, KV, T, B, pool.data.get_device())
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


def pages_read(pool, layer, table, rows, pos, check=False):
    """The keys and values that layer `layer` of the cache holds of n tokens: [n, 2, kv_heads, 256] for position pos[i] of
    sequence rows[i] of table (int32), in the pool's type, float16 for a pool in 4 bits (exactly the values that it
    stands for).  What is out of range gives zeros; check=True raises for it."""
    (B, width), n = table.shape, rows.shape[0]
    table, rows, pos = _ints(table, B, width), _ints(rows, n), _ints(pos, n)
    with _on(pool.data, table, rows, pos):
        out = torch.empty((n, 2, pool.kv_heads, pool.head_dim), device=table.device,
                          dtype=torch.float16 if pool.data.dtype is torch.uint8 else pool.data.dtype)
        L.check(L.lib().q35_pages_read(pool.desc(), layer, table.data_ptr(), width, B, rows.data_ptr(), pos.data_ptr(), n,
                                       out.data_ptr(), pool.status.data_ptr(), _stream()))
    if check:
        pool.check()
    return out


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


def beam_select(logits, scores, k, ended=None, check=False):
    """The next beams of G groups of W beams: logits [G, W, V] or [G * W, V] (float32, float16 or bfloat16), scores float32
    [G, W].  Of a group's continuations (beam w, token v), which score scores[g, w] + logits[g, w, v] - logsumexp of the
    row, the k highest: BeamSelect(scores float32, parents int32, tokens int32), all [G, k], highest first; among equal ones the
    lowest beam, in a beam the larger logit, then the lowest token.  parents are rows of the G * W, as pages_fork and states_fork take them.
    ended (int32 [G * W] or [G, W]; None: none): a beam with ended >= 0 goes on as it is, with that token.  A beam whose score
    is not finite has no continuation; a group with fewer than k is filled up with score -inf, parent -1, token -1.
    check=True synchronises and raises Q35Error (Q35_E_RANGE) for an ended token >= V, which leaves its beam without a
    continuation."""
    G, W = scores.shape
    V = logits.shape[-1]
    dtype, dev, f32, i32 = _DTYPES.get(logits.dtype), logits.device, torch.float32, torch.int32
    assert dtype is not None, logits.dtype
    assert scores.dtype is f32, scores.dtype
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    assert x.shape[0] == G * W, (tuple(logits.shape), tuple(scores.shape))
    if x.stride(1) != 1 or x.stride(0) < V:
        x = x.contiguous()
    scores = scores if scores.is_contiguous() else scores.contiguous()
    if ended is not None:
        ended = _ints(ended, *((G, W) if ended.dim() == 2 else (G * W,)))
    with _on(x, scores, ended):
        res = BeamSelect(torch.empty(G, k, dtype=f32, device=dev), torch.empty(G, k, dtype=i32, device=dev),
                         torch.empty(G, k, dtype=i32, device=dev))
        if G == 0:
            return res
        status = torch.zeros(1, dtype=i32, device=dev) if check else None
        nbytes = _beam_ws_bytes(G, W, V, k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        L.check(L.lib().q35_beam_select(x.data_ptr(), dtype, G, W, V, x.stride(0) if G * W > 1 else V, scores.data_ptr(), _ptr(ended), k,
                                        res.scores.data_ptr(), res.parents.data_ptr(), res.tokens.data_ptr(), _ptr(status), ws.data_ptr(),
                                        nbytes, _stream()))
        if check:
            L.check(L.lib().q35_status_check(status.data_ptr(), _stream()))
    return res


def states_fork(states, parents, out=None, check=False):
    """Row j of every tensor of `states` becomes what its row parents[j] was (int32 [B_out]; -1: row j stays), in place, or in
    the tensors of `out` (of the same rows, B_out of them).  The tensors [B, ...] have any type and a contiguous row; their rows
    may lie apart (a slice of a cache's tokens).  In place B_out is at most B.  The tensors must not overlap each other.
    Returns the tensors written.  check=True raises Q35Error (Q35_E_RANGE) for a parent outside [-1, B), which counts as -1."""
    states = list(states)
    dst = states if out is None else list(out)
    assert len(dst) == len(states), (len(dst), len(states))
    Bo = parents.shape[0]
    parents = _ints(parents, Bo)
    if not states or Bo == 0:
        return dst
    B, dev = states[0].shape[0], parents.get_device()
    assert B > 0 and (out is not None or Bo <= B), (Bo, B)
    # src, dst, src_stride, dst_stride, row_bytes of every state (one by one in ctypes' fields took 40 us for 36 states)
    flat = []
    for i, s in enumerate(states):
        assert s.shape[0] == B and s.get_device() == dev, "states of different rows, or on different devices"
        n, p = s.nbytes // B, s.data_ptr()
        ss = n if s.is_contiguous() else _row_stride(s, n)
        if out is None:
            flat += (p, p, ss, ss, n)
        else:
            d = dst[i]
            assert d.dtype is s.dtype and d.shape[1:] == s.shape[1:] and d.size(0) >= Bo, (tuple(s.shape), tuple(d.shape), Bo)
            assert d.get_device() == dev, "tensors on different devices"
            flat += (p, d.data_ptr(), ss, _row_stride(d, n), n)
    with _on(parents):
        status = torch.zeros(1, dtype=torch.int32, device=parents.device) if check else None
        L.check(L.lib().q35_states_fork(_words(len(flat)).pack(*flat), len(states), parents.data_ptr(), B, Bo, _ptr(status), _stream()))
        if check:
            L.check(L.lib().q35_status_check(status.data_ptr(), _stream()))
    return dst


@functools.lru_cache(maxsize=64)
def _words(n):
    return struct.Struct("=%dq" % n)


def _row_stride(t, row_bytes):
    """Bytes between the rows of t, whose own values must be contiguous."""
    if t.is_contiguous():
        return row_bytes
    assert t.shape[0] > 0 and t[0].is_contiguous() and t.stride(0) * t.element_size() >= row_bytes, (tuple(t.shape), t.stride())
    return t.stride(0) * t.element_size()

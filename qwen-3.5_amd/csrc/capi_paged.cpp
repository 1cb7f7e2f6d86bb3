// extern "C" entry points of the paged caches and the token scores.  Argument checking lives here;
// device-resident indices (pages, positions, parents, token ids) are checked by the kernels.
#include "pages.h"

#include <algorithm>
#include <cmath>

namespace q35 {
namespace {

inline hipStream_t S(void* s) { return static_cast<hipStream_t>(s); }
// No C++ exception (an error message that finds no memory) leaves a C entry point.
template <class F>
int entry(F&& f) {
  try {
    return f();
  } catch (...) {
    return Q35_E_NOMEM;
  }
}
inline bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return x < y + nb && y < x + na;
}
// A launch has fewer than 2^32 threads along x: so many blocks of 256.
constexpr int kMaxGrid = 1 << 24;
// The paged attention's append has one block for 4 (row, query or kv head)s and two more.
inline bool rows_fit(const q35_dims* d, int32_t T) { return (int64_t)T * (d->attn_heads + d->kv_heads) < (1 << 25); }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" {

int q35_status_check(uint32_t* status, void* stream) {
  return entry([&]() -> int {
    if (!status) return fail(Q35_E_ARG, "status_check: null pointer");
    uint32_t v = 0;
    Q35_HIP_TRY(hipMemcpyAsync(&v, status, sizeof(v), hipMemcpyDeviceToHost, S(stream)));
    Q35_HIP_TRY(hipStreamSynchronize(S(stream)));
    if (!v) return Q35_OK;
    const int rc = status_clear_launch(status, v, S(stream));
    if (rc) return rc;
    // (a bit that is set after this call has returned must not meet the clearing)
    Q35_HIP_TRY(hipStreamSynchronize(S(stream)));
    if (v & Q35_STATUS_ARG)
      return fail(Q35_E_RANGE, "a page, position, parent, token id or pair of pages was out of range or refused; the outputs it belongs to are invalid");
    return fail(Q35_E_NOMEM, "no free page left in the pool: entries of the page table were left -1");
  });
}

size_t q35_attention_paged_ws_bytes(const q35_dims* d, int32_t T, int32_t B) {
  if (!d || T < 1 || B < 1 || T > (1 << 20) || B > (1 << 20) || d->kv_heads < 1 || d->attn_heads < d->kv_heads ||
      d->attn_heads > kPageMaxHeads || d->attn_heads / d->kv_heads > kPageMaxRep || !rows_fit(d, T))
    return 0;
  return paged_attn_ws_bytes(d->attn_heads, d->kv_heads, T, B);
}

int q35_attention_core_paged(const q35_dims* d, q35_pages pool, int32_t layer, const float* q_gate, int32_t ld_qg,
                             const float* k_new, const float* v_new, int32_t kv_ld, int32_t T,
                             const int32_t* seq_start, const int32_t* pos, int32_t B, const int32_t* table,
                             int32_t ld_table, const float* q_norm, const float* k_norm, const float* rope_cos,
                             const float* rope_sin, int32_t rope_rows, float* out, int32_t ld_out, uint32_t* status,
                             void* ws, size_t ws_bytes, void* stream) {
  return entry([&]() -> int {
    int rc = check_pages(pool, "attention_paged");
    if (rc) return rc;
    if (!d || !q_gate || !k_new || !v_new || !seq_start || !pos || !table || !q_norm || !k_norm || !rope_cos || !rope_sin || !out)
      return fail(Q35_E_ARG, "attention_paged: null pointer");
    if (d->head_dim != kPageHd || pool.kv_heads != d->kv_heads)
      return fail(Q35_E_SHAPE, "attention_paged: head_dim must be 256 and the pool's kv heads the model's");
    if (d->kv_heads < 1 || d->attn_heads < 1 || d->attn_heads % d->kv_heads != 0 || d->attn_heads / d->kv_heads > kPageMaxRep ||
        d->attn_heads > kPageMaxHeads)
      return fail(Q35_E_SHAPE, "attention_paged: heads must be a multiple of kv heads, ratio <= 16, at most 1024");
    if (d->rot_dim < 2 || d->rot_dim > kPageHd || d->rot_dim % 2 != 0) return fail(Q35_E_SHAPE, "attention_paged: bad rotary dim");
    if (layer < 0 || layer >= pool.n_layers) return fail(Q35_E_SHAPE, "attention_paged: no such layer in the pool");
    if (T < 1 || B < 1 || T > (1 << 20) || B > (1 << 20) || ld_table < 1 || rope_rows < 1 || rope_rows > (1 << 30))
      return fail(Q35_E_SHAPE, "attention_paged: T and B in 1..2^20, ld_table >= 1 and rope_rows in 1..2^30 required");
    if (!rows_fit(d, T)) return fail(Q35_E_SHAPE, "attention_paged: T (heads + kv heads) < 2^25 required");
    if (ld_qg < 2 * d->attn_heads * kPageHd || kv_ld < d->kv_heads * kPageHd || ld_out < d->attn_heads * kPageHd)
      return fail(Q35_E_SHAPE, "attention_paged: row strides too small");
    if (ld_qg % 4 || kv_ld % 4 || ld_out % 4 || !aligned(q_gate, 16) || !aligned(k_new, 16) || !aligned(v_new, 16) ||
        !aligned(out, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16))
      return fail(Q35_E_ALIGN, "attention_paged: rows and norm weights must be 16-byte aligned");
    if (!ws || ws_bytes < q35_attention_paged_ws_bytes(d, T, B)) return fail(Q35_E_WS, "attention_paged: workspace too small");
    if (!aligned(ws, 16)) return fail(Q35_E_ALIGN, "attention_paged: workspace not 16-byte aligned");
    PagedAttn a;
    a.P = pool;
    a.layer = layer;
    a.nh = d->attn_heads; a.nkv = d->kv_heads; a.rot = d->rot_dim;
    a.T = T; a.B = B;
    a.ld_qg = ld_qg; a.ld_kv = kv_ld; a.ld_table = ld_table; a.ld_out = ld_out; a.rope_rows = rope_rows;
    a.eps = d->eps;
    a.scale = (float)(1.0 / std::sqrt((double)kPageHd));
    a.qg = q_gate; a.k = k_new; a.v = v_new; a.qnw = q_norm; a.knw = k_norm; a.rcos = rope_cos; a.rsin = rope_sin;
    a.start = seq_start; a.pos = pos; a.table = table;
    a.out = out;
    a.status = status;
    a.ws = ws;
    return paged_attn_launch(a, S(stream));
  });
}

size_t q35_pages_copy_ws_bytes(int32_t n) { return n <= kPageFewPairs ? 0 : (size_t)n; }

int q35_pages_copy(q35_pages src, q35_pages dst, const int32_t* src_ids, const int32_t* dst_ids, int32_t n,
                   uint32_t* status, void* ws, size_t ws_bytes, void* stream) {
  return entry([&]() -> int {
    int rc = check_pages(src, "pages_copy");
    if (!rc) rc = check_pages(dst, "pages_copy");
    if (rc) return rc;
    if (src.dtype != dst.dtype || src.n_layers != dst.n_layers || src.kv_heads != dst.kv_heads || src.page != dst.page)
      return fail(Q35_E_SHAPE, "pages_copy: the pools' pages differ in type, layers, heads or tokens");
    if (n < 0) return fail(Q35_E_SHAPE, "pages_copy: n must be >= 0");
    const size_t pb = page_bytes(src);
    const char *s0 = static_cast<const char*>(src.data), *d0 = static_cast<const char*>(dst.data);
    const char *s1 = s0 + pb * src.n_pages * src.n_layers, *d1 = d0 + pb * dst.n_pages * dst.n_layers;
    if (s0 == d0 ? src.n_pages != dst.n_pages : overlap(s0, s1 - s0, d0, d1 - d0))
      return fail(Q35_E_ARG, "pages_copy: two pools that overlap");
    if (n == 0) return Q35_OK;
    if (!src_ids || !dst_ids) return fail(Q35_E_ARG, "pages_copy: null pointer");
    if ((int64_t)n * (int64_t)(pb / 16384) >= kMaxGrid) return fail(Q35_E_SHAPE, "pages_copy: too many pages for one call");
    if (n > kPageFewPairs && (!ws || ws_bytes < q35_pages_copy_ws_bytes(n))) return fail(Q35_E_WS, "pages_copy: workspace too small");
    return pages_copy_launch(src, dst, src_ids, dst_ids, n, status, static_cast<uint8_t*>(ws), S(stream));
  });
}

int q35_pages_fork(q35_pages pool, const int32_t* table, int32_t ld_table, const int32_t* len, int32_t B,
                   const int32_t* parent, const int32_t* grow, int32_t B_out, int32_t* table_out, int32_t* len_out,
                   int32_t* refs, uint32_t* status, void* stream) {
  return entry([&]() -> int {
    const int rc = check_pages(pool, "pages_fork");
    if (rc) return rc;
    if (!table || !len || !parent || !table_out || !len_out || !refs) return fail(Q35_E_ARG, "pages_fork: null pointer");
    if (B < 1 || B > kPageMaxSeqs || B_out < 1 || B_out > kPageMaxSeqs || ld_table < 1 || ld_table > 65536)
      return fail(Q35_E_SHAPE, "pages_fork: 1..4096 rows of 1..65536 entries required");
    const size_t row = (size_t)ld_table * sizeof(int32_t);
    if ((int64_t)B_out * ld_table > kPageMaxEntries) return fail(Q35_E_SHAPE, "pages_fork: at most 2^26 entries");
    if (overlap(table, B * row, table_out, B_out * row)) return fail(Q35_E_ARG, "pages_fork: table_out must be another buffer");
    if (overlap(len, B * sizeof(int32_t), len_out, B_out * sizeof(int32_t))) return fail(Q35_E_ARG, "pages_fork: len_out must be another buffer");
    const size_t n = B_out * sizeof(int32_t);
    if (overlap(parent, n, len_out, n) || (grow && overlap(grow, n, len_out, n))) return fail(Q35_E_ARG, "pages_fork: len_out must be another buffer");
    ForkCall c;
    c.P = pool;
    c.table = table; c.len = len; c.parent = parent; c.grow = grow;
    c.ld = ld_table; c.B = B; c.Bo = B_out;
    c.table_out = table_out; c.len_out = len_out; c.refs = refs;
    c.status = status;
    return pages_fork_launch(c, S(stream));
  });
}

size_t q35_pages_compact_ws_bytes(int32_t n_pages) { return n_pages < 1 ? 0 : (2 * (size_t)n_pages + 1) * sizeof(int32_t); }

int q35_pages_compact(q35_pages pool, const int32_t* table, int32_t ld_table, int32_t B, int32_t* table_out,
                      int32_t* refs, int32_t* used, uint32_t* status, void* ws, size_t ws_bytes, void* stream) {
  return entry([&]() -> int {
    const int rc = check_pages(pool, "pages_compact");
    if (rc) return rc;
    if (!table || !table_out || !refs || !used) return fail(Q35_E_ARG, "pages_compact: null pointer");
    if (B < 1 || B > (1 << 20) || ld_table < 1 || ld_table > 65536)
      return fail(Q35_E_SHAPE, "pages_compact: 1..2^20 rows of 1..65536 entries required");
    const size_t ne = (size_t)B * ld_table;
    if (ne > (size_t)kPageMaxEntries) return fail(Q35_E_SHAPE, "pages_compact: at most 2^26 entries");
    if (overlap(table, ne * sizeof(int32_t), table_out, ne * sizeof(int32_t))) return fail(Q35_E_ARG, "pages_compact: table_out must be another buffer");
    if (!ws || ws_bytes < q35_pages_compact_ws_bytes(pool.n_pages)) return fail(Q35_E_WS, "pages_compact: workspace too small");
    if (!aligned(ws, 4)) return fail(Q35_E_ALIGN, "pages_compact: workspace not 4-byte aligned");
    CompactCall c;
    c.P = pool;
    c.table = table;
    c.ld = ld_table; c.B = B;
    c.table_out = table_out; c.refs = refs; c.used = used;
    c.status = status;
    c.moves = static_cast<int32_t*>(ws);
    return pages_compact_launch(c, S(stream));
  });
}

size_t q35_token_logprobs_ws_bytes(int32_t M, int32_t V, int32_t top) {
  if (M < 1 || V < 1 || top < 0 || top > kMaxTop) return 0;
  return std::max<size_t>(token_logprobs_ws_bytes(M, V, top), 256);
}

int q35_token_logprobs(const void* logits, int32_t dtype, int32_t M, int32_t V, int64_t ld, const int32_t* targets,
                       int32_t top, float* logprob, int32_t* rank, float* entropy, int32_t* top_ids,
                       float* top_logprobs, uint32_t* status, void* ws, size_t ws_bytes, void* stream) {
  return entry([&]() -> int {
    if (!logits || !entropy) return fail(Q35_E_ARG, "token_logprobs: null pointer");
    if (targets && (!logprob || !rank)) return fail(Q35_E_ARG, "token_logprobs: targets need logprob and rank");
    if (dtype != Q35_F32 && dtype != Q35_F16 && dtype != Q35_BF16) return fail(Q35_E_ARG, "token_logprobs: bad dtype");
    // (indices shifted by up to 8 values stay below 2^31)
    if (M < 1 || M >= kMaxGrid || V < 1 || V > (1 << 30) || ld < V) return fail(Q35_E_SHAPE, "token_logprobs: 1 <= M < 2^24, 1 <= V <= 2^30 and ld >= V required");
    if (top < 0 || top > kMaxTop || top > V) return fail(Q35_E_SHAPE, "token_logprobs: top must be in 0..64 and at most V");
    if (top > 0 && (!top_ids || !top_logprobs)) return fail(Q35_E_ARG, "token_logprobs: top needs top_ids and top_logprobs");
    if (!aligned(logits, elt_size(dtype))) return fail(Q35_E_ALIGN, "token_logprobs: logits not aligned to their type");
    if (!ws || ws_bytes < q35_token_logprobs_ws_bytes(M, V, top)) return fail(Q35_E_WS, "token_logprobs: workspace too small");
    if (!aligned(ws, 16)) return fail(Q35_E_ALIGN, "token_logprobs: workspace not 16-byte aligned");
    ScoreCall c;
    c.x = logits; c.dtype = dtype; c.M = M; c.V = V; c.top = top; c.ld = ld;
    c.targets = targets;
    c.logprob = logprob; c.rank = rank; c.entropy = entropy; c.top_ids = top_ids; c.top_lp = top_logprobs;
    c.status = status;
    c.ws = ws;
    return token_logprobs_launch(c, S(stream));
  });
}

}  // extern "C"

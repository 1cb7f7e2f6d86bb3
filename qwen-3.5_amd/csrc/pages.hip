// Pages of a cache: copies, forks, compaction.
//
// The bookkeeping of a fork or a compaction is whole-number work on a table of page numbers: a block does it by
// itself with a bitmap of the pool's pages in LDS, so that it needs no host round trip and no order among
// blocks; every choice (which page is new, which page moves where) is a rank among bits, hence the same on
// every run.  While the table is small, every block of one launch does it and then copies its share of the
// pages; else one block does it and a second launch copies.  A page of one layer is one contiguous run.
#include "pages.h"

#include <algorithm>

namespace q35 {

namespace {

constexpr int kCT = 256;        // threads of a copying block
constexpr int kUnit = 16384;    // bytes a block copies at a time: 4 x 16 bytes per thread (a page's last unit may have fewer)
constexpr int kPT = 1024;       // threads of a bookkeeping block
constexpr int kPW = kPT / 64;

// The `bytes` (a multiple of 16, kUnit at most) of a unit, by kCT threads, thread t of them
Q35_DEV void copy_unit(char* dst, const char* src, int t, int64_t bytes) {
  const int o = t * 16;
  if (bytes < kUnit) {
    for (int i = o; i < bytes; i += 16 * kCT) *reinterpret_cast<uint4*>(dst + i) = ldg16_nt(src + i);
    return;
  }
  uint4 v[kUnit / (16 * kCT)];
#pragma unroll
  for (int i = 0; i < kUnit / (16 * kCT); ++i) v[i] = ldg16_nt(src + o + i * 16 * kCT);
#pragma unroll
  for (int i = 0; i < kUnit / (16 * kCT); ++i) {
    const q35_u32x4 w = {v[i].x, v[i].y, v[i].z, v[i].w};
    __builtin_nontemporal_store(w, (Q35_GLOBAL q35_u32x4*)(dst + o + i * 16 * kCT));
  }
}

// (an atomic: calls on other streams may add bits at the same time)
__global__ void status_clear_kernel(uint32_t* status, uint32_t bits) {
  if (threadIdx.x == 0) __hip_atomic_fetch_and((Q35_GLOBAL uint32_t*)status, ~bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- copies
struct CopyArgs {
  char* src;
  char* dst;
  int64_t src_layer, dst_layer, page;  // bytes
  int32_t src_pages, dst_pages, same, n, units;
  const int32_t *sid, *did;
  const uint8_t* ok;  // nullptr: the block checks its pair itself
  uint32_t* status;
};

// Pair i is copied if both pages exist, no other pair names its destination and, in one pool, its
// destination is nobody's source and its source nobody's destination.
Q35_DEV bool pair_clash(int s, int d, int s2, int d2, int same) { return d2 == d || (same && (s2 == d || d2 == s)); }

// Blocks (pair i, layer, unit of the page).  Bound by HBM: 944 MB read and written in 178 us, 5.3 TB/s; 3 pages 3 us.
__global__ __launch_bounds__(kCT) void pages_copy_kernel(const CopyArgs a) {
  const int i = blockIdx.x / a.units, u = blockIdx.x % a.units, layer = blockIdx.y;
  const int s = a.sid[i], d = a.did[i];
  bool bad = (uint32_t)s >= (uint32_t)a.src_pages || (uint32_t)d >= (uint32_t)a.dst_pages;
  if (a.ok) {
    bad |= !a.ok[i];
  } else {
    bool clash = a.same && s == d;
    for (int j = threadIdx.x; j < a.n; j += kCT)
      if (j != i) clash |= pair_clash(s, d, a.sid[j], a.did[j], a.same);
    bad = __syncthreads_or(bad || clash);
  }
  if (bad) {
    if (threadIdx.x == 0 && u == 0 && layer == 0) raise_status(a.status, Q35_STATUS_ARG);
    return;
  }
  const int64_t o = (int64_t)u * kUnit;
  copy_unit(a.dst + layer * a.dst_layer + d * a.page + o, a.src + layer * a.src_layer + s * a.page + o, threadIdx.x, a.page - o);
}

// ok[i] for many pairs: bitmaps of the pages that are a source, a destination, a destination twice.
__global__ __launch_bounds__(kPT) void pages_copy_check_kernel(const CopyArgs a, uint8_t* ok) {
  extern __shared__ uint32_t bm[];
  const int ws = (a.src_pages + 31) / 32, wd = (a.dst_pages + 31) / 32;
  uint32_t *S = bm, *D = bm + ws, *DD = D + wd;
  for (int e = threadIdx.x; e < ws + 2 * wd; e += kPT) bm[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kPT) {
    const int s = a.sid[i], d = a.did[i];
    if ((uint32_t)s < (uint32_t)a.src_pages) atomicOr(&S[s >> 5], 1u << (s & 31));
    if ((uint32_t)d < (uint32_t)a.dst_pages) {
      const uint32_t b = 1u << (d & 31);
      if (atomicOr(&D[d >> 5], b) & b) atomicOr(&DD[d >> 5], b);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kPT) {
    const int s = a.sid[i], d = a.did[i];
    bool good = (uint32_t)s < (uint32_t)a.src_pages && (uint32_t)d < (uint32_t)a.dst_pages;
    if (good) {
      good = !((DD[d >> 5] >> (d & 31)) & 1u);
      if (a.same) good = good && !((S[d >> 5] >> (d & 31)) & 1u) && !((D[s >> 5] >> (s & 31)) & 1u);
    }
    ok[i] = good ? 1 : 0;
  }
}

// ---- rows as values
// A wave per (token, plane and head), 4 values a lane.  Bound by its round trips (ids, table, row): 2.2 us for one
// token, 4.7 for 33 of long contexts.
__global__ __launch_bounds__(kCT) void pages_read_kernel(const ReadCall c) {
  const int lane = threadIdx.x & 63, planes = 2 * c.P.kv_heads;
  const int64_t item = (int64_t)blockIdx.x * (kCT / 64) + (threadIdx.x >> 6), i = item / planes;
  if (i >= c.n) return;
  const int ph = (int)(item - i * planes), b = c.row[i], p = c.pos[i];
  int page = -1;
  if ((uint32_t)b < (uint32_t)c.B && p >= 0 && p < (int64_t)c.ld * c.P.page) page = c.table[(int64_t)b * c.ld + p / c.P.page];
  const bool ok = (uint32_t)page < (uint32_t)c.P.n_pages;
  if (!ok && lane == 0) raise_status(c.status, Q35_STATUS_ARG);
  const int rb = row_bytes(c.P);
  const char* r = static_cast<const char*>(c.P.data);
  if (ok) r += ((int64_t)c.layer * c.P.n_pages + page) * (int64_t)page_bytes(c.P) + ((int64_t)ph * c.P.page + (p & (c.P.page - 1))) * rb;
  if (c.P.dtype == Q35_F32) {
    const uint4 v = ok ? reinterpret_cast<const uint4*>(r)[lane] : make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(c.out)[item * 64 + lane] = v;
    return;
  }
  uint2 v = make_uint2(0, 0);
  if (ok && c.P.dtype != Q35_Q4) v = reinterpret_cast<const uint2*>(r)[lane];
  if (ok && c.P.dtype == Q35_Q4) {
    const uint32_t code = reinterpret_cast<const uint16_t*>(r)[lane], word = reinterpret_cast<const uint16_t*>(r + kPageHd / 2)[lane >> 3];
    const float s = (float)__builtin_bit_cast(_Float16, (uint16_t)(word & 0xFFF0u));
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      h[j] = __builtin_bit_cast(uint16_t, (_Float16)(s * (float)((int)(code >> (4 * j) & 15) - (int)(word & 15))));
    v = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  }
  reinterpret_cast<uint2*>(c.out)[item * 64 + lane] = v;
}

// ---- block-wide helpers of the bookkeeping kernels
// exclusive sum of v over the block's threads; *total = the sum.  sh: kPW ints.
Q35_DEV int block_excl(int v, int* sh, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sh[w] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPW; ++i) {
    before += i < w ? sh[i] : 0;
    all += sh[i];
  }
  *total = all;
  return before + x - v;
}

// before[w] = bits set in the words before w; returns the number of all.  Every thread holds a run of words.
Q35_DEV int count_before(const uint32_t* bits, int* before, int words, int* sh) {
  const int per = (words + kPT - 1) / kPT;
  const int w0 = min(words, (int)threadIdx.x * per), w1 = min(words, w0 + per);
  int cnt = 0;
  for (int w = w0; w < w1; ++w) cnt += __popc(bits[w]);
  int n;
  int r = block_excl(cnt, sh, &n);
  for (int w = w0; w < w1; ++w) {
    before[w] = r;
    r += __popc(bits[w]);
  }
  __syncthreads();
  return n;
}

// ---- fork
// The parent of row j and its length; -1 for an empty row or a refused parent
Q35_DEV int fork_parent(const ForkCall& c, int j, int* n, bool* bad) {
  const int p = c.parent[j];
  *n = 0;
  *bad = p < -1 || p >= c.B;
  if (*bad || p < 0) return -1;
  const int l = c.len[p];
  if (l < 0 || l > (int64_t)c.ld * c.P.page) {
    *bad = true;
    return -1;
  }
  *n = l;
  return p;
}

// The first `tail` tokens of page src to page dst, in one (layer, plane and head), by a block of nt threads; pages
// outside the pool are left alone
Q35_DEV void copy_tail(const ForkCall& c, int part, int src, int dst, int tail, int nt) {
  if (src == dst || (uint32_t)src >= (uint32_t)c.P.n_pages || (uint32_t)dst >= (uint32_t)c.P.n_pages) return;
  const int rb = row_bytes(c.P), planes = 2 * c.P.kv_heads;
  const int64_t head = (int64_t)c.P.page * rb, pb = head * planes;
  const int layer = part / planes, ph = part - layer * planes;
  char* base = static_cast<char*>(c.P.data) + (int64_t)layer * c.P.n_pages * pb + ph * head;
  const char* f = base + src * pb;
  char* t = base + dst * pb;
  for (int o = threadIdx.x * 16; o < tail * rb; o += nt * 16) {
    const uint4 v = ldg16(f + o);
    *reinterpret_cast<uint4*>(t + o) = v;
  }
}

// LDS of the bookkeeping, in ints
struct ForkLds {
  int words, first, len, par, base, tail, refs, fresh, total;
};
// Counts of up to this many pages are kept in LDS (64 KB); a shared prefix's counts, added to from every
// row, otherwise wait for each other in the cache (that case: 15.8 us, 10.5 so).
constexpr int kLdsRefs = 16384;
constexpr int kMoved = -2;  // (-1: an entry outside the pool)
__host__ __device__ inline ForkLds fork_lds(int n_pages, int B, int Bo, bool one) {
  ForkLds L;
  L.words = (n_pages + 31) / 32;
  L.first = 2 * L.words;      // [words] pages that a kept entry names, [words] pages in use before the word
  L.len = L.first + B;        // parent -> its first child
  L.par = L.len + Bo;         // row -> its length
  L.base = L.par + Bo;        // row -> its parent
  L.tail = L.base + Bo + 1;   // row -> new pages before it
  L.refs = L.tail + Bo;       // row -> the partly filled page that it keeps (kMoved: none)
  L.fresh = L.refs + (n_pages <= kLdsRefs ? n_pages : 0);  // row -> its first new page, if the launch copies too
  L.total = L.fresh + (one ? Bo : 0);
  return L;
}

// Every step spreads its entries over all threads (a wave per row waited for its row's loads in turn: 35
// instead of 17 us for 200 rows of 36 entries).
// Bound by its round trips and block-wide steps: 8 rows 7.6 us with the copies, 200 rows of 36 entries 10 without.  One
// block's rate bounds large tables: 33 rows of 4097 entries, 29000 pages in use, 78 us, 132000 in use 250.
// kOne: any number of blocks, which all do the bookkeeping, each for itself; the first writes it down, and then each
// copies its share of the last pages' tokens.  That saves a launch, and a wait for it.
// A partly filled page may be appended to, so one row may name it: the first that continues it, if no row names it as a
// full page (as where a sequence was cut back into a prefix that others hold).  The rows' claims meet in the counts,
// which are 0 for a page that no full entry names: the largest wins, whatever the order.
template <bool kOne>
__global__ __launch_bounds__(kPT) void pages_fork_kernel(const ForkCall c) {
  extern __shared__ int lds[];
  __shared__ int sh[kPW];
  const int tid = threadIdx.x, np = c.P.n_pages, page = c.P.page, shift = __ffs(page) - 1;  // (a power of two)
  const ForkLds L = fork_lds(np, c.B, c.Bo, kOne);
  const int words = L.words;
  const bool lead = !kOne || blockIdx.x == 0;
  uint32_t* bits = reinterpret_cast<uint32_t*>(lds);
  int *before = lds + words, *first = lds + L.first, *len = lds + L.len, *par = lds + L.par, *base = lds + L.base;
  int *tail = lds + L.tail, *fresh = lds + L.fresh;
  bool bad = false;
  for (int e = tid; e < words; e += kPT) bits[e] = 0;
  int* refs = lds + L.refs;
  const bool counted = np <= kLdsRefs;
  for (int e = tid; e < np; e += kPT) (counted ? refs : c.refs)[e] = 0;
  for (int e = tid; e < c.B; e += kPT) first[e] = INT32_MAX;
  __syncthreads();
  for (int j = tid; j < c.Bo; j += kPT) {
    int n;
    bool b;
    const int p = fork_parent(c, j, &n, &b);
    if (p >= 0) atomicMin(&first[p], j);
    if (lead) c.len_out[j] = n;
    len[j] = n;
    par[j] = p;
    tail[j] = kMoved;
    if (kOne) fresh[j] = -1;
    bad |= b;
  }
  __syncthreads();
  // full pages, -1 behind them; a parent's partly filled page goes to its first child, which may keep it
  const int ne = c.Bo * c.ld;  // (at most 2^26)
  constexpr int kU = 4;  // entries of a thread in flight
  for (int e0 = tid; e0 < ne; e0 += kU * kPT) {
    int v[kU], kind[kU], row[kU];  // kind: 0 none, 1 behind the row's full pages, 2 full, 3 partly filled
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const int x = min(e0 + i * kPT, ne - 1);
      const int j = x / c.ld, e = x - j * c.ld, n = len[j], full = n >> shift;
      kind[i] = e < full ? 2 : e == full && (n & (page - 1)) != 0 && first[par[j]] == j ? 3 : 1;
      if (e0 + i * kPT >= ne) kind[i] = 0;
      v[i] = kind[i] >= 2 ? c.table[(int64_t)par[j] * c.ld + e] : -1;
      row[i] = j;
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      if (kind[i] == 0) continue;
      if (kind[i] >= 2 && (uint32_t)v[i] >= (uint32_t)np) {
        v[i] = -1;
        bad = true;
      }
      if (kind[i] == 3) {
        tail[row[i]] = v[i];
        v[i] = -1;
      } else if (v[i] >= 0) {
        atomicOr(&bits[v[i] >> 5], 1u << (v[i] & 31));
        if (lead) {
          if (counted) atomicAdd(&refs[v[i]], 1);
          else __hip_atomic_fetch_add((Q35_GLOBAL int32_t*)&c.refs[v[i]], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
      if (lead) c.table_out[e0 + i * kPT] = v[i];
    }
  }
  __syncthreads();
  // claims of 2 and more, the lowest row's the largest; the page's count is then 1, its owner's
  for (int j = tid; j < c.Bo; j += kPT) {
    const int v = tail[j];
    if (v < 0) continue;
    if ((bits[v >> 5] >> (v & 31)) & 1u) tail[j] = kMoved;
    else if (counted) atomicMax(&refs[v], c.Bo + 1 - j);
    else __hip_atomic_fetch_max((Q35_GLOBAL int32_t*)&c.refs[v], c.Bo + 1 - j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  for (int j = tid; j < c.Bo; j += kPT) {
    const int v = tail[j];
    if (v < 0) continue;
    const int won = counted ? __hip_atomic_load(&refs[v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)
                            : __hip_atomic_load((Q35_GLOBAL int32_t*)&c.refs[v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (won != c.Bo + 1 - j) {
      tail[j] = kMoved;
      continue;
    }
    if (counted) __hip_atomic_store(&refs[v], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    else __hip_atomic_store((Q35_GLOBAL int32_t*)&c.refs[v], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    atomicOr(&bits[v >> 5], 1u << (v & 31));
    if (lead) c.table_out[(int64_t)j * c.ld + (len[j] >> shift)] = v;
  }
  __syncthreads();
  // entries that row j keeps
  auto kept_of = [&](int j) { return (len[j] >> shift) + (tail[j] != kMoved ? 1 : 0); };
  int run = 0;  // new pages of the rows before this group of kPT
  for (int j0 = 0; j0 < c.Bo; j0 += kPT) {
    const int j = j0 + tid;
    int need = 0;
    if (j < c.Bo) {
      int64_t g = c.grow ? c.grow[j] : 0;
      if (g < 0) {
        g = 0;
        bad = true;
      }
      int64_t total = ((int64_t)len[j] + g + page - 1) >> shift;
      if (total > c.ld) {
        total = c.ld;
        bad = true;
      }
      need = (int)total - kept_of(j);
    }
    int all;
    const int b = block_excl(need, sh, &all);
    if (j < c.Bo) base[j] = run + b;
    run += all;
  }
  if (tid == 0) base[c.Bo] = run;
  __syncthreads();
  const int used = count_before(bits, before, words, sh);
  // the r-th free page is the r-th new entry (where pages are short, the last entries stay -1)
  auto place = [&](int r, int page_id) {
    int lo = 0, hi = c.Bo;  // the row j with base[j] <= r < base[j + 1]
    while (hi - lo > 1) {
      const int m = (lo + hi) / 2;
      if (base[m] <= r) lo = m;
      else hi = m;
    }
    if (lead) c.table_out[(int64_t)lo * c.ld + kept_of(lo) + r - base[lo]] = page_id;
    if (kOne && r == base[lo]) fresh[lo] = page_id;
  };
  for (int p = tid; p < np; p += kPT) {
    const uint32_t w = bits[p >> 5], below = (1u << (p & 31)) - 1u;
    const int r = p - (before[p >> 5] + __popc(w & below));
    const bool dealt = !((w >> (p & 31)) & 1u) && r < run;
    if (dealt) place(r, p);
    if (counted) {
      if (lead) c.refs[p] = dealt ? 1 : refs[p];
    } else if (dealt) {
      c.refs[p] = 1;
    }
  }
  if (bad && lead) raise_status(c.status, Q35_STATUS_ARG);
  if (tid == 0 && lead && run > np - used) raise_status(c.status, Q35_STATUS_FULL);
  if constexpr (kOne) {
    __syncthreads();
    const int planes = 2 * c.P.kv_heads, parts = c.P.n_layers * planes;
    for (int i = blockIdx.x; i < c.Bo * parts; i += gridDim.x) {
      const int j = i / parts, p = par[j], n = len[j];
      // (a row that keeps its last page has no copy: its first new page, if any, is behind its tokens)
      if (p < 0 || (n & (page - 1)) == 0 || tail[j] != kMoved) continue;
      copy_tail(c, i - j * parts, c.table[(int64_t)p * c.ld + (n >> shift)], fresh[j], n & (page - 1), kPT);
    }
  }
}

// The tokens of last pages that were not kept: blocks (row j, layer, plane and head).  4728 copies of 19 KB from 3
// sequences' pages, which the caches hold: 18 us, 5 TB/s written.
__global__ __launch_bounds__(kCT) void pages_fork_copy_kernel(const ForkCall c) {
  const int j = blockIdx.x;
  int n;
  bool b;
  const int p = fork_parent(c, j, &n, &b);
  const int tail = n % c.P.page;
  if (p < 0 || tail == 0) return;
  const int at = n / c.P.page;
  copy_tail(c, blockIdx.y * gridDim.z + blockIdx.z, c.table[(int64_t)p * c.ld + at], c.table_out[(int64_t)j * c.ld + at], tail, kCT);
}

// ---- compaction
// Unit e of (move, layer, part of a page of pb bytes) by kCT threads
Q35_DEV void copy_move(const CompactCall& c, const int32_t* holes, const int32_t* movers, int64_t e, int64_t pb, int units, int t) {
  const int u = (int)(e % units), layer = (int)(e / units % c.P.n_layers);
  const int m = (int)(e / units / c.P.n_layers);
  char* base = static_cast<char*>(c.P.data) + (int64_t)layer * c.P.n_pages * pb + (int64_t)u * kUnit;
  copy_unit(base + holes[m] * pb, base + movers[m] * pb, t, pb - (int64_t)u * kUnit);
}
// kOne: as pages_fork_kernel's; the lists of moves stay in LDS.  514 MB read and written in 101 us, 5.1 TB/s (HBM); a
// small pool 5.6 us (round trips).  Larger tables are one block's, a load of a thread at a time, each entry twice: 33
// rows of 4097 entries 99 us with 29000 pages in use, 265 with 132000, beside what moves.
template <bool kOne>
__global__ __launch_bounds__(kPT) void pages_compact_kernel(const CompactCall c, int64_t pb, int units) {
  extern __shared__ uint32_t bits[];  // pages in use, then the number of them before each word, then the moves
  __shared__ int sh[kPW];
  const int tid = threadIdx.x;
  const int np = c.P.n_pages, words = (np + 31) / 32;
  int* before = reinterpret_cast<int*>(bits + words);
  int32_t* holes = kOne ? before + words : c.moves;  // at most half of the pages move
  int32_t* movers = holes + (kOne ? np / 2 : np);
  const int64_t ne = (int64_t)c.B * c.ld;
  const bool lead = !kOne || blockIdx.x == 0;
  bool bad = false;
  for (int e = tid; e < words; e += kPT) bits[e] = 0;
  if (lead)
    for (int e = tid; e < np; e += kPT) c.refs[e] = 0;
  __syncthreads();
  for (int64_t e = tid; e < ne; e += kPT) {
    const int v = c.table[e];
    if ((uint32_t)v < (uint32_t)np) atomicOr(&bits[v >> 5], 1u << (v & 31));
    else bad |= v != -1;
  }
  __syncthreads();
  const int n = count_before(bits, before, words, sh);
  auto rank = [&](int p) { return before[p >> 5] + __popc(bits[p >> 5] & ((1u << (p & 31)) - 1u)); };  // pages in use < p
  const int low = n < np ? rank(n) : n;  // pages in use below n; n - low of them move
  // hole h (the h-th unused page below n) and mover h (the h-th page in use from n on)
  for (int p = tid; p < np; p += kPT) {
    const bool live = (bits[p >> 5] >> (p & 31)) & 1u;
    const int k = rank(p);
    if (p < n && !live) holes[p - k] = p;
    if (p >= n && live) movers[k - low] = p;
  }
  if (tid == 0 && lead) *c.used = n;
  __syncthreads();
  if (lead) {
    for (int64_t e = tid; e < ne; e += kPT) {
      int v = c.table[e];
      if ((uint32_t)v >= (uint32_t)np) v = -1;
      else {
        if (v >= n) v = holes[rank(v) - low];
        __hip_atomic_fetch_add((Q35_GLOBAL int32_t*)&c.refs[v], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      c.table_out[e] = v;
    }
    if (bad) raise_status(c.status, Q35_STATUS_ARG);
  }
  if constexpr (kOne) {
    const int64_t all = (int64_t)(n - low) * c.P.n_layers * units;
    constexpr int kG = kPT / kCT;
    for (int64_t e = (int64_t)blockIdx.x * kG + tid / kCT; e < all; e += (int64_t)gridDim.x * kG)
      copy_move(c, holes, movers, e, pb, units, tid % kCT);
  } else {
    // the copying launch reads the number of moves behind the lists
    if (tid == 0) c.moves[2 * (int64_t)np] = n - low;
  }
}

// Any number of blocks: units of (move, layer, part of the page) dealt round.
__global__ __launch_bounds__(kCT) void pages_compact_copy_kernel(const CompactCall c, int64_t pb, int units) {
  const int np = c.P.n_pages;
  const int64_t all = (int64_t)c.moves[2 * (int64_t)np] * c.P.n_layers * units;
  for (int64_t e = blockIdx.x; e < all; e += gridDim.x) copy_move(c, c.moves, c.moves + np, e, pb, units, threadIdx.x);
}

// One launch does everything (kOne) while the table is small, since every block reads it, and the pool's counts or
// moves fit LDS: 8 beams 8.6 -> 7.7 us in a graph, 15.5 -> 12.6 called alone; 20 sequences compacted 22.0 -> 20.3,
// 40 of 4000 tokens 307 -> 291.  A fork must have few copies besides: blocks of 1024 threads take one at a time (64
// rows of 24 copies each 12.7 us as two launches, 13.0 as one; 200 rows 28 and 36).
constexpr int kOneEntries = 16384;
constexpr int kOneCopies = 4;  // per CU

}  // namespace

int check_pages(const q35_pages& P, const char* what) {
  auto no = [&](int code, const char* why) { return fail(code, std::string(what) + why); };
  if (!P.data) return no(Q35_E_ARG, ": null pool");
  if (P.dtype != Q35_F32 && P.dtype != Q35_F16 && P.dtype != Q35_BF16 && P.dtype != Q35_Q4) return no(Q35_E_ARG, ": bad pool dtype");
  if (P.head_dim != kPageHd) return no(Q35_E_SHAPE, ": head_dim must be 256");
  if (P.page < 16 || P.page > 256 || (P.page & (P.page - 1)) != 0)
    return no(Q35_E_SHAPE, ": tokens per page must be a power of two in 16..256");
  if (P.n_layers < 1 || P.n_layers > 65535 || P.n_pages < 1 || P.n_pages > kPageMaxPages || P.kv_heads < 1 || P.kv_heads > 1024)
    return no(Q35_E_SHAPE, ": layers, pages (at most 262144) and kv heads (at most 1024) must be positive");
  if ((reinterpret_cast<uintptr_t>(P.data) & 15) != 0) return no(Q35_E_ALIGN, ": pool not 16-byte aligned");
  return Q35_OK;
}

int status_clear_launch(uint32_t* status, uint32_t bits, hipStream_t st) {
  hipLaunchKernelGGL(status_clear_kernel, dim3(1), dim3(64), 0, st, status, bits);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

int pages_copy_launch(const q35_pages& src, const q35_pages& dst, const int32_t* sid, const int32_t* did, int n,
                      uint32_t* status, uint8_t* ok, hipStream_t st) {
  CopyArgs a;
  const int64_t pb = (int64_t)page_bytes(src);
  a.src = static_cast<char*>(src.data);
  a.dst = static_cast<char*>(dst.data);
  a.page = pb;
  a.src_layer = pb * src.n_pages;
  a.dst_layer = pb * dst.n_pages;
  a.src_pages = src.n_pages;
  a.dst_pages = dst.n_pages;
  a.same = src.data == dst.data;
  a.n = n;
  a.units = (int)((pb + kUnit - 1) / kUnit);
  a.sid = sid;
  a.did = did;
  a.status = status;
  a.ok = nullptr;
  if (n > kPageFewPairs) {
    const size_t lds = ((src.n_pages + 31) / 32 + 2 * (size_t)((dst.n_pages + 31) / 32)) * 4;
    allow_lds<pages_copy_check_kernel>(lds);
    hipLaunchKernelGGL(pages_copy_check_kernel, dim3(1), dim3(kPT), lds, st, a, ok);
    Q35_HIP_TRY(hipGetLastError());
    a.ok = ok;
  }
  hipLaunchKernelGGL(pages_copy_kernel, dim3(n * a.units, src.n_layers), dim3(kCT), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

int pages_read_launch(const ReadCall& c, hipStream_t st) {
  const int64_t items = (int64_t)c.n * 2 * c.P.kv_heads;
  hipLaunchKernelGGL(pages_read_kernel, dim3((uint32_t)((items + kCT / 64 - 1) / (kCT / 64))), dim3(kCT), 0, st, c);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

int pages_fork_launch(const ForkCall& c, hipStream_t st) {
  const int64_t parts = (int64_t)c.Bo * c.P.n_layers * 2 * c.P.kv_heads;
  const bool one = c.P.n_pages <= kLdsRefs && c.Bo * c.ld <= kOneEntries && parts <= kOneCopies * device_cus();
  const size_t lds = (size_t)fork_lds(c.P.n_pages, c.B, c.Bo, one).total * 4;
  if (one) {
    allow_lds<pages_fork_kernel<true>>(lds);
    hipLaunchKernelGGL(pages_fork_kernel<true>, dim3((uint32_t)std::min<int64_t>(parts, device_cus())), dim3(kPT), lds, st, c);
    Q35_HIP_TRY(hipGetLastError());
    return Q35_OK;
  }
  allow_lds<pages_fork_kernel<false>>(lds);
  hipLaunchKernelGGL(pages_fork_kernel<false>, dim3(1), dim3(kPT), lds, st, c);
  Q35_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(pages_fork_copy_kernel, dim3(c.Bo, c.P.n_layers, 2 * c.P.kv_heads), dim3(kCT), 0, st, c);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

int pages_compact_launch(const CompactCall& c, hipStream_t st) {
  const int words = (c.P.n_pages + 31) / 32;
  const int64_t pb = (int64_t)page_bytes(c.P);
  const int units = (int)((pb + kUnit - 1) / kUnit);
  // at most half of the pages move
  const int64_t most = (int64_t)(c.P.n_pages / 2) * c.P.n_layers * units;
  const int64_t ne = (int64_t)c.B * c.ld;
  constexpr int kG = kPT / kCT;
  if (c.P.n_pages <= kLdsRefs && ne <= kOneEntries) {
    const size_t lds = (size_t)words * 8 + (size_t)(c.P.n_pages / 2) * 8;
    allow_lds<pages_compact_kernel<true>>(lds);
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>((most + kG - 1) / kG, device_cus()));
    hipLaunchKernelGGL(pages_compact_kernel<true>, dim3((uint32_t)grid), dim3(kPT), lds, st, c, pb, units);
    Q35_HIP_TRY(hipGetLastError());
    return Q35_OK;
  }
  allow_lds<pages_compact_kernel<false>>((size_t)words * 8);
  hipLaunchKernelGGL(pages_compact_kernel<false>, dim3(1), dim3(kPT), (size_t)words * 8, st, c, pb, units);
  Q35_HIP_TRY(hipGetLastError());
  const int grid = (int)(most < 1 ? 1 : most > 8 * device_cus() ? 8 * device_cus() : most);
  hipLaunchKernelGGL(pages_compact_copy_kernel, dim3(grid), dim3(kCT), 0, st, c, pb, units);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

}  // namespace q35

// Attention of new tokens over a paged cache: q/k RMSNorm (1 + w), rotary, append of keys and values to
// the sequences' pages, causal softmax(q K^T / 16) V with shared kv heads, sigmoid output gate.
//
// Launches: append (with the plan), the attention of the sequences with few new tokens, that of the
// sequences with many (either left out where paged_layout says that no sequence needs it), and the join of what
// the plan cut.
#include "pages.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace q35 {

namespace {

constexpr int kHd = kPageHd;
constexpr int kT = 256;

// Sequence b: its rows, and whether they lie in the call's rows and their positions in the table and the
// rotary rows.
struct Seq {
  int b, s0, n, p0;  // sequence, first row, rows, tokens cached before
};
Q35_DEV bool load_seq(const PagedAttn& a, int b, Seq* s) {
  s->b = b;
  s->s0 = a.start[b];
  const int s1 = a.start[b + 1];
  s->n = s1 - s->s0;
  s->p0 = a.pos[b];
  const int64_t cap = (int64_t)a.ld_table * a.P.page;
  const int64_t lim = cap < a.rope_rows ? cap : a.rope_rows;
  return s->s0 >= 0 && s1 >= s->s0 && s1 <= a.T && s->p0 >= 0 && (int64_t)s->p0 + s->n <= lim;
}
// The sequence of the wave's row t: b with start[b] <= t < start[b + 1]; false if there is none or it is
// refused.  The lanes look at 64 starts at a time.
Q35_DEV bool find_seq(const PagedAttn& a, int t, Seq* s) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = a.B;  // the last b in [lo, lo + len) with start[b] <= t
  while (len > 1) {
    const int step = (len + 63) / 64, off = lane * step;
    const int c = __popcll(__ballot(off < len && a.start[lo + min(off, len - 1)] <= t));
    if (c == 0) return false;
    lo += (c - 1) * step;
    len = min(step, len - (c - 1) * step);
  }
  return load_seq(a, lo, s) && t >= s->s0 && t < s->s0 + s->n;
}

// ------------------------------------------------------------------ the plan
// Work is dealt out in units of 32 cached tokens of one kv head for one tile of query rows, laid end to
// end over all tiles of all sequences: block g of G takes the units [g W / G, (g + 1) W / G), whatever
// tiles they belong to.  So ragged batches load every CU alike, and a few long sequences are split as
// finely as many short ones are not.  Where a block's range cuts a tile, it leaves (max, sum, output)
// of its part, and paged_join_kernel joins the parts; only the first and the last tile of a block can be
// cut, so two slots per block hold them all.
// A part of a second tile costs a block its queries, first loads and join once more, up to 6 us over a cache in 4 bits: there
// "few" blocks take a part of one tile alone if that comes out even enough (kCutUnits).
//
// Two kinds of tiles: sequences of few rows ("few": the cache's stream bounds them) and chunks ("many":
// the matrix cores do).
constexpr int kUnit = 32;       // tokens of a unit
constexpr int kFewRows = 16;    // query rows (token, head) of a "few" tile
constexpr int kManyRows = 128;  // of a "many" tile

// All that a block needs to know of a tile, in one load
struct alignas(16) Tile {
  int64_t u0;                       // its first unit
  int32_t units, b, i, s0, n, p0;   // units per kv head; sequence, tile of it, its first row, rows, cached tokens
};
// The plan of one kind: block g starts at unit g q + min(g, r)
struct PlanHead {
  int64_t w, q;  // units of all tiles
  int32_t r, tiles, blocks;
  int32_t whole;  // 0, or q: a (tile, kv head) is laid out over a multiple of that many units, so no block has parts of two
};

struct AttnArgs {
  PagedAttn c;
  int32_t page_shift;     // log2 of the tokens per page
  int32_t rep, tok_many;  // query heads per kv head; tokens of a "many" tile
  uint32_t rep_inv;
  int32_t few_most;       // sequences of at most this many new tokens are "few"
  int32_t max_tiles[2], max_blocks[2], part_rows[2];
  PlanHead* head;        // [2]
  int64_t* once;         // units of "few" that no other tile reads
  float* q;              // [T][heads][256] queries after norm and rotary
  float* qmax;           // [T][heads] largest |value|
  int32_t* tile0;        // [2][B] first tile of the sequence in the list of each kind
  Tile* tiles[2];
  int4* cut;             // [T][heads] where the parts of a cut tile lie (cut_record)
  float* part_ml[2];     // [2 max_blocks][part_rows][2]
  float* part_o[2];      // [2 max_blocks][part_rows][256]
};

Q35_DEV int kind_of(const AttnArgs& A, int n) { return n <= A.few_most ? 0 : 1; }
// x / rep for x < 2^28 (rep_inv = 2^32 / rep + 1)
Q35_DEV int div_rep(const AttnArgs& A, int x) { return A.rep == 1 ? x : (int)__umulhi((uint32_t)x, A.rep_inv); }
Q35_DEV int tiles_of(const AttnArgs& A, int n) {
  if (n <= 0) return 0;
  return kind_of(A, n) ? (n + A.tok_many - 1) / A.tok_many : (n * A.rep + kFewRows - 1) / kFewRows;
}
// cached tokens that tile i of the sequence looks at
Q35_DEV int tile_len(const AttnArgs& A, const Seq& s, int i) {
  const int tok = kind_of(A, s.n) ? (i + 1) * A.tok_many - 1 : div_rep(A, (i + 1) * kFewRows - 1);
  return s.p0 + min(tok, s.n - 1) + 1;
}
// units that a (tile, kv head) of n units is laid out over
Q35_DEV int laid_out(int n, int whole) { return whole ? (int)((uint32_t)(n + whole - 1) / (uint32_t)whole) * whole : n; }
// first unit of block g, and the block that holds unit u
Q35_DEV int64_t block_u0(const PlanHead& h, int g) { return h.q * g + min(g, h.r); }
Q35_DEV int unit_block(const PlanHead& h, int64_t u) {
  const int64_t big = h.r * (h.q + 1);  // the first r blocks take q + 1 units
  const int64_t x = u < big ? u : u - h.r, y = u < big ? h.q + 1 : h.q;
  int64_t g = (int64_t)((float)x * __builtin_amdgcn_rcpf((float)y));  // (at most 512: off by one at most)
  if (g * y > x) --g;
  else if ((g + 1) * y <= x) ++g;
  return (int)g;
}

// exclusive sum over the block's kT threads
template <class V>
Q35_DEV V plan_excl(V v, V* sh, V* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  V x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sh[w] = x;
  __syncthreads();
  V before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; ++i) {
    before += i < w ? sh[i] : 0;
    all += sh[i];
  }
  *total = all;
  return before + x - v;
}

// Blocks take whole parts while the longest has at most kCutUnits more than an even share (both ways, us of a call among others: 40
// tokens behind 2048 .. 4096, 16 and 17 units, 37.0 and 35.2; 12 x 5 behind 2730 .. 8191, 20 and 21, 39.5 and 37.6; 60 of one
// token behind 8000, 59 and 63, 76 and 76; 33 behind 16000, 65 and 72, 78.8 and 79.8; 90 behind 4000, 45 and 63, 60.5 and 70.5), times the
// tiles that an even share may have parts of (two prompts of 500 tokens, 8 and 16, tiles of 1 to 16: 83 and 40).
constexpr int kCutUnits = 4;
constexpr int kWholeMost = 1 << 22;  // units (quotients are estimated in f32)
// The units of a block if each of `most` blocks at most takes a part of one (tile, kv head) alone: the fewest from `even` on, the even
// share, with which the blocks are enough for all tiles (one a thread, of `units` for each kv head); 0 if that is none of
// the first 64, or too many.  Lane c of each wave tries even + c over a quarter of the tiles.
Q35_DEV int whole_units(int units, int tiles, int nkv, int even, int most) {
  __shared__ int n[kT], sum[kT / 64][64], least[kT / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  n[threadIdx.x] = units;
  __syncthreads();
  const int per = even + lane;
  const float inv = 1.f / (float)per;
  int blocks = 0, low = n[0];
  for (int x = w; x < tiles; x += kT / 64) {
    int k = (int)((float)n[x] * inv);  // (off by one at most: units and quotients are below 2^22)
    k += (k + 1) * per <= n[x] ? 1 : k * per > n[x] ? -1 : 0;
    blocks += k + (k * per < n[x] ? 1 : 0);
    low = min(low, n[x]);
  }
  sum[w][lane] = blocks;
  least[w] = low;
  __syncthreads();
  blocks = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; ++i) {
    blocks += sum[i][lane];
    low = min(low, least[i]);
  }
  const unsigned long long fits = __ballot(blocks <= most / nkv);
  const int more = fits ? __builtin_ctzll(fits) : 64;
  return more < 64 && more <= kCutUnits * max(1, even / low) ? even + more : 0;
}

// Made by one block: the sequences' tiles, then each tile's first unit.  kWhole: "few" blocks may take whole parts.
template <bool kWhole>
Q35_DEV void make_plan(const AttnArgs& A) {
  const PagedAttn& a = A.c;
  __shared__ int si[kT / 64];
  __shared__ int64_t sl[kT / 64];
  // (up to kT sequences stay in LDS: their tiles' search and a second look at them were trips through memory)
  __shared__ int first[2][kT];
  __shared__ Seq seqs[kT];
  const int tid = threadIdx.x;
  const bool held = a.B <= kT;
  int count[2] = {0, 0};
  bool bad = false, falls = false;
  for (int b0 = 0; b0 < a.B; b0 += kT) {
    const int b = b0 + tid;
    int nt[2] = {0, 0};
    if (b < a.B) {
      Seq s;
      if (load_seq(a, b, &s)) nt[kind_of(A, s.n)] = tiles_of(A, s.n);
      else bad = true;
      falls |= s.n < 0;
      if (held) seqs[b] = s;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int all;
      const int t = plan_excl(nt[k], si, &all);
      if (b < a.B) {
        if (held) first[k][b] = count[k] + t;
        else A.tile0[(int64_t)k * a.B + b] = count[k] + t;
      }
      count[k] += all;
    }
  }
  if (bad) raise_status(a.status, Q35_STATUS_ARG);
  // (starts that fall could name more rows than there are: nothing is done then)
  if (__syncthreads_or(falls)) count[0] = count[1] = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int nt = min(count[k], A.max_tiles[k]);
    auto tile0 = [&](int b) { return held ? first[k][b] : A.tile0[(int64_t)k * a.B + b]; };
    int64_t run = 0, laid = 0;
    int whole = 0;
    for (int x0 = 0; x0 < nt; x0 += kT) {
      const int x = x0 + tid;
      Tile t = {0, 0, 0, 0, 0, 0, 0};
      if (x < nt) {
        // the last sequence with tile0 <= x: those without tiles of this kind share the next one's number
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
          const int m = (lo + hi) / 2;
          if (tile0(m) <= x) lo = m;
          else hi = m;
        }
        Seq s;
        if (held) s = seqs[lo];
        else load_seq(a, lo, &s);
        t.b = lo;
        t.i = x - tile0(lo);
        t.units = (tile_len(A, s, t.i) + kUnit - 1) / kUnit;
        t.s0 = s.s0;
        t.n = s.n;
        t.p0 = s.p0;
      }
      int64_t all;
      t.u0 = run + plan_excl((int64_t)t.units * a.nkv, sl, &all);
      run += all;
      laid = run;
      if (kWhole && k == 0 && nt <= kT && nt * a.nkv <= A.max_blocks[0] && run <= (int64_t)kWholeMost) {
        // (a step of each wave at least: it takes as long as one wave's, and there are fewer parts to join: one token behind 8000
        // 21.9 -> 16.8 us of a call, 100 x 2 tokens behind 120 24.8 -> 18.0)
        const int even = max(kT / 64, (int)((run + A.max_blocks[0] - 1) / A.max_blocks[0]));
        whole = whole_units(t.units, nt, a.nkv, even, A.max_blocks[0]);
        if (whole) {
          t.u0 = plan_excl((int64_t)laid_out(t.units, whole) * a.nkv, sl, &laid);
        }
      }
      if (x < nt) A.tiles[k][x] = t;
    }
    if (tid == 0) {
      // (a "many" block takes four units at least: what it leaves to the join costs about one)
      const int64_t least = k ? 4 : 1, most = (run + least - 1) / least;
      const int64_t blocks = most < A.max_blocks[k] ? most : A.max_blocks[k];
      A.head[k] = whole ? PlanHead{run, whole, 0, nt, (int)(laid / whole), whole}
                        : PlanHead{run, blocks ? run / blocks : 0, blocks ? (int)(run % blocks) : 0, nt, (int)blocks, 0};
    }
  }
}

// Made by another block: the units of "few" that one tile alone reads, all but what lies in pages that the sequence
// before has at the same place (looked at in eight places) and what a sequence's second tile reads.
Q35_DEV void count_once(const AttnArgs& A) {
  const PagedAttn& a = A.c;
  __shared__ int64_t sl[kT / 64];
  if (A.max_blocks[0] == 0) return;
  int64_t once = 0;
  for (int b = threadIdx.x; b < a.B; b += kT) {
    Seq s;
    if (!load_seq(a, b, &s) || s.n == 0 || kind_of(A, s.n) != 0) continue;
    const int ctx = s.p0 + s.n, pages = ((ctx - 1) >> A.page_shift) + 1;
    const int32_t* row = a.table + (int64_t)b * a.ld_table;
    int own = 8;
    if (b > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t c = (2 * i + 1) * (int64_t)pages >> 4;
        own -= row[c] == row[c - a.ld_table] ? 1 : 0;
      }
    }
    once += (int64_t)((ctx + kUnit - 1) / kUnit) * a.nkv * own / 8;
  }
  int64_t all;
  plan_excl(once, sl, &all);
  if (threadIdx.x == 0) *A.once = all;
}

template <int DT>
struct Elt;
template <>
struct Elt<Q35_F32> {
  typedef float T;
};
template <>
struct Elt<Q35_F16> {
  typedef _Float16 T;
};
template <>
struct Elt<Q35_BF16> {
  typedef __bf16 T;
};
template <>
struct Elt<Q35_Q4> {
  typedef uint8_t T;  // (bytes)
};

template <int DT>
constexpr int kRow = DT == Q35_Q4 ? kQ4Row : kHd;  // elements of a token's row
template <int DT>
Q35_DEV int64_t plane_elts(const PagedAttn& a) { return (int64_t)a.nkv * a.P.page * kRow<DT>; }
template <int DT>
Q35_DEV int64_t page_elts(const PagedAttn& a) { return 2 * plane_elts<DT>(a); }

// wave sum in f64, the same in every lane
Q35_DEV double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// what one lane of a wave wrote to LDS is read by others of the same wave
Q35_DEV void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// A key's value as the cache holds it: rounded to f32, then to the cache's type (both to nearest even).
// The empty asm keeps the compiler from rounding f64 to f16 in one step, as it otherwise does.
template <class E>
Q35_DEV E stored(double y) {
  float f = (float)y;
  asm("" : "+v"(f));
  return (E)f;
}

// ------------------------------------------------------------------ 4 bits
// A row of a Q35_Q4 cache: a code c of 4 bits per value, and for each 32 values a word: an f16 scale s of 7 significant
// bits (the word without its low 4 bits) and a zero z (those); the value is s (c - z).  |c - z| has 4 bits, so a value
// is exactly an f16, and the kernels multiply f16 values, as over f16 caches, with nothing lost in between.
// lo = min(0, the least value), hi = max(0, the largest), s the smallest such number that is not below
// (hi - lo) / 15, z = lo / -s and c = y / s + z, both quotients rounded to nearest even: a value is off by s / 2 at
// most.  (7 bits: s is at most 1/64 larger than it need be.)
//
// y / s to the nearest whole number, ties to even (|y| <= 16 s, s of 7 significant bits): an estimate, put right by its remainder, which
// is exact (near a whole multiple of s the difference is).
Q35_DEV float quot_even(float y, float s, float inv) {
  float q = __builtin_rintf(y * inv);
  const float e = __builtin_fmaf(-q, s, y), h = 0.5f * s;
  const bool odd = (int)q & 1;
  q += e > h || (e == h && odd) ? 1.f : e < -h || (e == -h && odd) ? -1.f : 0.f;
  return q;
}
// The codes of the lane's 4 values (a group of 32 is that of 8 lanes), and the group's word
Q35_DEV uint32_t quantise4(const float (&in)[4], uint32_t& word) {
  float y[4], lo = 0.f, hi = 0.f;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    fine = fine && fabsf(in[j]) < INFINITY;
    y[j] = fminf(fmaxf(in[j], -32768.f), 32768.f);
    lo = fminf(lo, y[j]);
    hi = fmaxf(hi, y[j]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, 64));
    hi = fmaxf(hi, __shfl_xor(hi, o, 64));
  }
  const unsigned long long odd = __ballot(!fine) >> (threadIdx.x & 56);
  if (odd & 0xff) {  // a value that is no number, or infinite: none of the group's is
    word = 0x7FF0;
    return 0;
  }
  const double x = ((double)hi - (double)lo) / 15.0;
  uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)(float)x) & 0xFFF0u;
  if ((double)(float)__builtin_bit_cast(_Float16, (uint16_t)b) < x) b += 16;
  const float s = (float)__builtin_bit_cast(_Float16, (uint16_t)b);
  if (b == 0) {
    word = 0;
    return 0;
  }
  const float inv = 1.f / s, z = quot_even(-lo, s, inv);
  word = b | (uint32_t)z;
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) c |= (uint32_t)fminf(fmaxf(quot_even(y[j], s, inv) + z, 0.f), 15.f) << (4 * j);
  return c;
}
// 4 values of a group's keys or values as f16 pairs.  1024 + c and 64 + c are the bits 0x6400 | c and 0x5400 | c << 4; their
// differences from 1024 + z and 64 + z are exact, and so is the product with s.
struct Word2 {  // of two groups, in halves
  uint32_t s, n0, n4;  // s, -(1024 + z), -(64 + z)
};
Q35_DEV Word2 word2(uint32_t w) {
  const uint32_t z = w & 0x000F000Fu;
  return Word2{w & 0xFFF0FFF0u, z | 0xE400E400u, z << 4 | 0xD400D400u};
}
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
Q35_DEV uint32_t value2(uint32_t c, uint32_t n, uint32_t s) {
  return __builtin_bit_cast(uint32_t, (h2)((__builtin_bit_cast(h2, c) + __builtin_bit_cast(h2, n)) * __builtin_bit_cast(h2, s)));
}
// The masks in scalar registers and the exponents in vector ones: one instruction ands and ors then (constants would be
// literals of two).
struct Nibbles {
  uint32_t m0, m4, e0, e4;
};
Q35_DEV Nibbles nibbles() {
  Nibbles c = {0x000F000Fu, 0x00F000F0u, 0x64006400u, 0x54005400u};
  asm("" : "+s"(c.m0), "+s"(c.m4), "+v"(c.e0), "+v"(c.e4));
  return c;
}
Q35_DEV uint32_t low_nibbles(uint32_t t, const Word2& w, const Nibbles& c) { return value2((t & c.m0) | c.e0, w.n0, w.s); }
Q35_DEV uint32_t high_nibbles(uint32_t t, const Word2& w, const Nibbles& c) { return value2((t & c.m4) | c.e4, w.n4, w.s); }
// 8 values (one dword of codes) as operands: values p and p + 4 in the halves of word p
Q35_DEV q35_u32x4 values8(uint32_t t, const Word2& w, const Nibbles& c) {
  const uint32_t d = t >> 8;
  return q35_u32x4{low_nibbles(t, w, c), high_nibbles(t, w, c), low_nibbles(d, w, c), high_nibbles(d, w, c)};
}

// Keys and values of the new tokens into their pages, and the normalised, rotated queries (with each one's
// largest |value|) into the workspace; a wave per (row, kv head or query head).  Blocks 0 and 1 make the plan.  Bound by
// its chain of round trips (starts, table, stores) while rows are few: 4.3 us for one token, 17.6 for 2048.
template <int DT>
__global__ __launch_bounds__(kT) void paged_append_kernel(const AttnArgs A) {
  typedef typename Elt<DT>::T E;
  const PagedAttn& a = A.c;
  __shared__ double xs[kT / 64][kHd];
  if (blockIdx.x < 2) {
    if (blockIdx.x == 0) make_plan<DT == Q35_Q4>(A);
    else count_once(A);
    return;
  }
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, per = a.nkv + a.nh;
  const int64_t item = ((int64_t)blockIdx.x - 2) * (kT / 64) + wid;
  const int64_t t = item / per;
  const int hd = (int)(item % per), g = hd, h = hd - a.nkv;  // kv head g, or query head h
  if (t >= a.T) return;
  // (the row's values are asked for before its sequence is known: it lies in the call's rows either way)
  const int d = 4 * lane, half = a.rot / 2;
  const bool query = h >= 0;
  const float4 in = *reinterpret_cast<const float4*>(query ? a.qg + t * a.ld_qg + (int64_t)h * 2 * kHd + d
                                                           : a.k + t * a.ld_kv + (int64_t)g * kHd + d);
  const float4 w = *reinterpret_cast<const float4*>((query ? a.qnw : a.knw) + d);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (query) {
    if (lane == 0) A.cut[t * a.nh + h] = make_int4(0, 0, 0, 0);
  } else {
    v = *reinterpret_cast<const float4*>(a.v + t * a.ld_kv + (int64_t)g * kHd + d);
  }
  Seq s;
  if (!find_seq(a, (int)t, &s)) return;
  const int p = s.p0 + (int)t - s.s0;
  const float* cs = a.rcos + (int64_t)p * a.rot;
  const float* sn = a.rsin + (int64_t)p * a.rot;
  if (query) {
    float* x = reinterpret_cast<float*>(xs[wid]);
    const float r = rsqrt_f(wave_sum(in.x * in.x + in.y * in.y + in.z * in.z + in.w * in.w) / (float)kHd + a.eps);
    float y[4] = {in.x * r * (1.0f + w.x), in.y * r * (1.0f + w.y), in.z * r * (1.0f + w.z), in.w * r * (1.0f + w.w)};
    *reinterpret_cast<float4*>(x + d) = make_float4(y[0], y[1], y[2], y[3]);
    wave_lds_sync();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = d + j;
      if (i < a.rot) y[j] = y[j] * cs[i] + (i < half ? -x[i + half] : x[i - half]) * sn[i];
    }
    const int64_t o = t * a.nh + h;
    *reinterpret_cast<float4*>(A.q + o * kHd + d) = make_float4(y[0], y[1], y[2], y[3]);
    float m = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
    for (int e = 32; e > 0; e >>= 1) m = fmaxf(m, __shfl_xor(m, e, 64));
    if (lane == 0) A.qmax[o] = m;
    return;
  }
  const int page = a.table[(int64_t)s.b * a.ld_table + (p >> A.page_shift)];
  if ((uint32_t)page >= (uint32_t)a.P.n_pages) {
    if (lane == 0) raise_status(a.status, Q35_STATUS_ARG);
    return;
  }
  const double x0 = in.x, x1 = in.y, x2 = in.z, x3 = in.w;
  const double r = 1.0 / sqrt(wave_sum64((x0 * x0 + x1 * x1) + (x2 * x2 + x3 * x3)) / (double)kHd + (double)a.eps);
  double y[4] = {x0 * r * (1.0 + (double)w.x), x1 * r * (1.0 + (double)w.y), x2 * r * (1.0 + (double)w.z), x3 * r * (1.0 + (double)w.w)};
  double* x = xs[wid];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[d + j] = y[j];
  wave_lds_sync();
  E* kr = static_cast<E*>(a.P.data) + ((int64_t)a.layer * a.P.n_pages + page) * page_elts<DT>(a) +
          ((int64_t)g * a.P.page + (p & (a.P.page - 1))) * kRow<DT>;
  E* vr = kr + plane_elts<DT>(a);
  const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = d + j;
    if (i < a.rot) y[j] = y[j] * (double)cs[i] + (i < half ? -x[i + half] : x[i - half]) * (double)sn[i];
  }
  if constexpr (DT == Q35_Q4) {
    const float kk[4] = {(float)y[0], (float)y[1], (float)y[2], (float)y[3]};
    uint32_t kw, vw;
    const uint32_t kc = quantise4(kk, kw), vc = quantise4(vv, vw);
    *reinterpret_cast<uint16_t*>(kr + 2 * lane) = (uint16_t)kc;
    *reinterpret_cast<uint16_t*>(vr + 2 * lane) = (uint16_t)vc;
    if ((lane & 7) == 0) {
      *reinterpret_cast<uint16_t*>(kr + kHd / 2 + lane / 4) = (uint16_t)kw;
      *reinterpret_cast<uint16_t*>(vr + kHd / 2 + lane / 4) = (uint16_t)vw;
    }
  } else {
    E ko[4], vo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ko[j] = stored<E>(y[j]);
      vo[j] = (E)vv[j];
    }
    typedef E E4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<E4*>(kr + d) = E4{ko[0], ko[1], ko[2], ko[3]};
    *reinterpret_cast<E4*>(vr + d) = E4{vo[0], vo[1], vo[2], vo[3]};
  }
}

// ------------------------------------------------------------------ shared by the attention kernels
typedef float f4 __attribute__((ext_vector_type(4)));

Q35_DEV float max_x32(float v) {  // the larger of lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
Q35_DEV float max_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
Q35_DEV float add_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
Q35_DEV float add_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
Q35_DEV Tile load_tile(const Tile* p) {  // (two 16-byte loads; a copy of the structure goes through private memory)
  const int4 a = reinterpret_cast<const int4*>(p)[0], b = reinterpret_cast<const int4*>(p)[1];
  Tile t;
  t.u0 = (int64_t)a.y << 32 | (uint32_t)a.x;
  t.units = a.z; t.b = a.w; t.i = b.x; t.s0 = b.y; t.n = b.z; t.p0 = b.w;
  return t;
}

// The same in every lane: in scalar registers
Q35_DEV int64_t uniform(int64_t v) {
  const int lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)hi << 32 | (uint32_t)lo;
}
Q35_DEV Tile uniform(Tile t) {
  t.u0 = uniform(t.u0);
  t.units = __builtin_amdgcn_readfirstlane(t.units);
  t.b = __builtin_amdgcn_readfirstlane(t.b);
  t.i = __builtin_amdgcn_readfirstlane(t.i);
  t.s0 = __builtin_amdgcn_readfirstlane(t.s0);
  t.n = __builtin_amdgcn_readfirstlane(t.n);
  t.p0 = __builtin_amdgcn_readfirstlane(t.p0);
  return t;
}

// The block's first tile, the one that holds unit u: every thread looks at some (they are few).  The first
// ones are asked for before the plan's head has arrived.
struct Start {
  Tile t;
  int x;
};
template <bool kWhole>
Q35_DEV bool block_start(const AttnArgs& A, int k, PlanHead* head, Start* sh) {
  const int x0 = threadIdx.x;
  Tile t;
  if (x0 < A.max_tiles[k]) t = load_tile(&A.tiles[k][x0]);
  *head = A.head[k];
  if ((int)blockIdx.x >= head->blocks) return false;
  const int64_t u = block_u0(*head, blockIdx.x);
  for (int x = x0; x < head->tiles; x += blockDim.x) {
    if (x != x0) t = load_tile(&A.tiles[k][x]);
    if (t.u0 <= u && u < t.u0 + (int64_t)(kWhole ? laid_out(t.units, head->whole) : t.units) * A.c.nkv) {
      sh->t = t;
      sh->x = x;
    }
  }
  __syncthreads();
  return true;
}

// Where the parts of a cut tile lie: block g's slots are 2 g (its first segment) and 2 g + 1.  Written for the part
// that holds the tile's first unit u0: its slot + 1 (0: not cut), the row in its slots (-1 - row for "many"),
// the tile's last unit.
Q35_DEV int4 cut_record(int slot, int row, int64_t u0, int units) {
  const int64_t last = u0 + units - 1;
  return make_int4(slot + 1, row, (int)(uint32_t)last, (int)(last >> 32));
}

// Page of tokens j0 .. (16 of them share one); pages outside the pool count as page 0.  The table is read
// through the constant address space and j0 is the wave's: a scalar load, which waits for nothing else (as a
// vector load it waited for every key and value under way).
Q35_DEV int page_of(const AttnArgs& A, const int32_t* row, int j0, bool* bad) {
  const PagedAttn& a = A.c;
  typedef __attribute__((address_space(4))) const int32_t cint;
  const int v = ((cint*)row)[__builtin_amdgcn_readfirstlane(j0 >> A.page_shift)];
  if ((uint32_t)v < (uint32_t)a.P.n_pages) return v;
  *bad = true;
  return 0;
}

// ------------------------------------------------------------------ few new tokens
// A block takes one tile - up to 16 rows (token, query head) of a kv head - over some units; its 4 waves
// take every 4th unit, each with its own running softmax, and are joined at the end.
//
// The keys of a unit go from the cache straight into the operand registers of S^T = K Q^T (keys in rows,
// query rows in columns), its values into those of O^T += V^T P^T: the scores come out where the weights
// are needed as operands, a row's maximum and sum stay in its lanes, and nothing passes LDS between the
// two products.  The order of the summed index is free as long as both operands share it: with 16-bit
// caches the k-slot (lane group g, j) of the second product (16x16x32) stands for key 4 g + j (j < 4) or
// 16 + 4 g + j - 4, the lanes that hold those scores, and a value row's 16-byte pieces are dealt to
// lanes so that each holds 8 keys of the same 8 dims, which a byte permute turns into operands.  f32
// caches are multiplied in f32 (16x16x4).
// A query value and a weight are carried whole, as 2 f16 or 3 bf16 parts with a product each; the matrix
// cores have time for that: the bound is the cache's stream.
// A block's first unit waits for the instructions too: code that runs once is fetched at about 64 bytes
// in 35 ns, so the loops' bodies are kept short.
// Bound by the stream of the cache: 33 tokens over 958 MB of bf16 170 us, 5.6 TB/s (a kernel with the same loads
// and nothing else 6.0); one token behind 517 in f32 8.0 us, round trips.
template <int DT>
Q35_DEV f4 mma(q35_u32x4 x, q35_u32x4 y, f4 c) {
  if constexpr (DT == Q35_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(q35_b8, x), __builtin_bit_cast(q35_b8, y), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(q35_h8, x), __builtin_bit_cast(q35_h8, y), c, 0, 0, 0);
}
// y -> f16 halves (hi, lo), both to nearest: y = hi + lo to 2^-24 of y, or 2^-25 where that is more (f16's last
// subnormal step).  What is left over has either sign; rounded toward zero it would add up over a context.
Q35_DEV void split2_near(float y0, float y1, uint32_t& hi, uint32_t& lo) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 h = __builtin_convertvector((f2{y0, y1}), h2);
  const h2 l = __builtin_convertvector((f2{y0 - (float)h[0], y1 - (float)h[1]}), h2);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}
constexpr int kFewLd = kHd + 4;
constexpr int kFewLds = 4 * kFewRows * kFewLd * 4;
// 4 bits: the queries' operands, then each wave's rows: keys of 16 tokens, of 16 more, and their values
constexpr int kQ4Half = 16 * kQ4Row;
constexpr int kQ4Rows = 2 * 8 * 64 * 16;
static_assert(kQ4Rows + 4 * 4 * kQ4Half <= kFewLds);

template <bool kStream>
Q35_DEV q35_u32x4 ldg_if(const void* p) {
  if constexpr (kStream) return __builtin_nontemporal_load((const Q35_GLOBAL q35_u32x4*)p);
  else return *(const Q35_GLOBAL q35_u32x4*)p;
}
// os: the queries' operands, then the waves' outputs [wave][row][kFewLd]
template <int DT, bool kStream>
Q35_DEV void few_run(const AttnArgs& A, const PlanHead& H, const Start& sh, float* os, float (&ms)[4][kFewRows],
                     float (&ls)[4][kFewRows]) {
  typedef typename Elt<DT>::T E;
  constexpr bool kWide = DT == Q35_F32, k4 = DT == Q35_Q4, kHalf = DT == Q35_F16 || k4;
  constexpr int kQ = kWide ? 1 : kHalf ? 2 : 3;  // parts of a query or weight
  constexpr int kW = kWide ? 2 : 1;                       // 16-byte words of 8 values
  constexpr int kH = kWide ? 1 : 2, kS = 16 * kH;          // keys of a wave's step
  // how far (log2) a score may pass the running maximum before the sums are rescaled (64 multiplications; in most of the first
  // steps some row has a new maximum): 4 bits' weights are f16 of 2^15 at most then (calls, us: 33 tokens behind 16000 80.1 -> 78.3,
  // 60 behind 8000 77.2 -> 75.5, 40 behind 2048 .. 4096 36.0 -> 35.2).
  constexpr float kSlack = k4 ? 3.f : 0.f;
  const PagedAttn& a = A.c;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  int64_t u = uniform(block_u0(H, blockIdx.x));
  const int64_t u_end = uniform(block_u0(H, blockIdx.x + 1));
  Tile t = uniform(load_tile(&sh.t));
  int x = sh.x;
  const float sl2 = a.scale * 1.44269504088896341f;
  q35_u32x4* const qs = reinterpret_cast<q35_u32x4*>(os);  // [part][step][lane]
  const Nibbles nib = nibbles();
  bool bad = false;
  // 4 bits: unpacking bounds (of about 710 vector instructions for 32 tokens 128 for each of and / or, subtracting z and multiplying by
  // s; with s z taken off the sums instead, 100 fewer, more registers and no faster).  Of a SIMD's two waves the older one then goes first, and the
  // younger ends alone; a wave that is further through its steps has a lower priority (calls, us: 33 tokens behind 16000 80.9 ->
  // 78.3, behind 20000 96.2 -> 94.3; short streams as they were).
  const int quarter = max(1, (int)((u_end - u) >> 4));  // of a wave's steps
  int left = 4 * quarter;
  if constexpr (k4) __builtin_amdgcn_s_setprio(3);
#pragma unroll 1
  for (int seg = 0; u < u_end; ++seg) {
    int gk = 0;
    int64_t off = u - t.u0;
    const int laid = k4 ? laid_out(t.units, H.whole) : t.units;
    for (; off >= laid; off -= laid) ++gk;
    const int k0 = (int)off, k1 = (int)min((int64_t)t.units, k0 + (u_end - u));
    const int rows = min(kFewRows, t.n * A.rep - t.i * kFewRows);
    const int pr = t.i * kFewRows + min(n, rows - 1), tok = div_rep(A, pr), h = gk * A.rep + pr - tok * A.rep;
    const int lim = t.p0 + tok;   // the last token the lane's row sees (rows past the last one repeat it)
    const int end = t.p0 + t.n;   // tokens from here on do not exist
    const int32_t* row = a.table + (int64_t)t.b * a.ld_table;
    const E* base = static_cast<const E*>(a.P.data) + (int64_t)a.layer * a.P.n_pages * page_elts<DT>(a) + (int64_t)gk * a.P.page * kRow<DT>;
    // pages of the step's 16-key halves
    auto pages = [&](int j0, int& pa, int& pb) {
      pa = page_of(A, row, j0, &bad);
      pb = kH == 1 || a.P.page > 16 || j0 + 16 >= end ? pa : page_of(A, row, j0 + 16, &bad);
    };
    q35_u32x4 kr[k4 ? 1 : kH][8 * kW], vr[k4 ? 1 : 4 * kH][2 * kW];
    auto load_k = [&](int j0, int pa, int pb) {
#pragma unroll
      for (int hf = 0; hf < kH; ++hf) {
        const int slot = (j0 + 16 * hf + n) & (a.P.page - 1);
        const E* p = base + (int64_t)(hf ? pb : pa) * page_elts<DT>(a) + (int64_t)slot * kHd + (kWide ? 4 : 8) * g;
#pragma unroll
        for (int i = 0; i < 8 * kW; ++i) kr[hf][i] = ldg_if<kStream>(p + (kWide ? 16 : 32) * i);
      }
    };
    auto load_v = [&](int j0, int pa, int pb) {
#pragma unroll
      for (int hf = 0; hf < kH; ++hf) {
        const int slot = (j0 + 16 * hf + 4 * g) & (a.P.page - 1);  // 4 keys of one page
        const E* p = base + plane_elts<DT>(a) + (int64_t)(hf ? pb : pa) * page_elts<DT>(a) + (int64_t)slot * kHd + (kWide ? 4 : 8) * n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int w = 0; w < 2 * kW; ++w) vr[4 * hf + j][w] = ldg_if<kStream>(p + j * kHd + w * (128 / kW));
      }
    };
    // 4 bits: the rows of 16 tokens are one run of 2304 bytes, which passes LDS: read piece by piece into the
    // operands' places, every line was asked for three times, and the L1 waited for it half of the time (33 tokens over
    // 400 MB 104 us, 94 so).  st[8]: the runs' last 256 bytes, a quarter of the wave each.
    q35_u32x4 st[9];
    char* const rows_lds = reinterpret_cast<char*>(os) + kQ4Rows + wid * 4 * kQ4Half;
    auto load_rows = [&](int j0, int pa, int pb) {
      const E* ka = base + (int64_t)pa * page_elts<DT>(a) + (int64_t)(j0 & (a.P.page - 1)) * kRow<DT>;
      const E* kb = base + (int64_t)pb * page_elts<DT>(a) + (int64_t)((j0 + 16) & (a.P.page - 1)) * kRow<DT>;
      const E* from[4] = {ka, kb, ka + plane_elts<DT>(a), kb + plane_elts<DT>(a)};
#pragma unroll
      for (int i = 0; i < 8; ++i) st[i] = ldg_if<kStream>(from[i >> 1] + (i & 1) * 1024 + 16 * lane);
      st[8] = ldg_if<kStream>((g < 2 ? g == 0 ? from[0] : from[1] : g == 2 ? from[2] : from[3]) + 2048 + 16 * n);
    };
    auto store_rows = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) *(q35_u32x4*)(rows_lds + (i >> 1) * kQ4Half + (i & 1) * 1024 + 16 * lane) = st[i];
      *(q35_u32x4*)(rows_lds + g * kQ4Half + 2048 + 16 * n) = st[8];
    };
    // queries: column n; dims 32 st + 8 g .. (16-bit), 16 st + 4 g .. (f32); each wave lays out a quarter.  They are
    // asked for first: loads arrive in order, and the operands can be laid out while keys and values are under way
    // (one token behind 517: 8.6 -> 8.0 us).
    const int64_t qi = (int64_t)(t.s0 + tok) * a.nh + h;
    f4 qv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qv[i] = *(const Q35_GLOBAL f4*)(A.q + qi * kHd + (kWide ? 16 * (4 * wid + i) + 4 * g
                                                          : k4 ? 64 * g + 8 * (2 * wid + (i >> 1)) + 4 * (i & 1)
                                                               : 32 * (2 * wid + (i >> 1)) + 8 * g + 4 * (i & 1)));
    float qm = 0.f;
    if constexpr (kHalf) qm = A.qmax[qi];
    int j0 = k0 * kUnit + wid * kS, pa = 0, pb = 0;
    const int j1 = min(k1 * kUnit, end);
    if (j0 < j1) {
      pages(j0, pa, pb);
      if constexpr (k4) {
        load_rows(j0, pa, pb);
      } else {
        load_k(j0, pa, pb);
        load_v(j0, pa, pb);
      }
    }
    float qscale = sl2;
    {
      float fq = 1.f;
      if constexpr (kHalf) {  // a power of two per query brings its largest value to 2^14
        float inv;
        split_scale(qm, fq, inv);
        qscale = sl2 * inv;
      }
#pragma unroll
      for (int i = 0; i < 2 * kW; ++i) {
        const int st = 2 * kW * wid + i;
        if constexpr (kWide) {
          qs[st * 64 + lane] = __builtin_bit_cast(q35_u32x4, qv[i]);
        } else {
          const f4 v0 = qv[2 * i], v1 = qv[2 * i + 1];
          const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
          q35_u32x4 qb[3];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t p0, p1, p2 = 0;
            if constexpr (k4) split2_near(v[j] * fq, v[j + 4] * fq, p0, p1);  // (values8's order)
            else if constexpr (kHalf) split2_near(v[2 * j] * fq, v[2 * j + 1] * fq, p0, p1);
            else split3(v[2 * j], v[2 * j + 1], p0, p1, p2);
            qb[0][j] = p0;
            qb[1][j] = p1;
            qb[2][j] = p2;
          }
#pragma unroll
          for (int q = 0; q < kQ; ++q) qs[(q * 8 + st) * 64 + lane] = qb[q];
        }
      }
    }
    __syncthreads();
    f4 o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    // A step waits for its keys, then its values, while the next step's are under way: that takes a loop whose every
    // step loads, and a last step apart (at a load that only some steps make, the compiler waits for all: 33 tokens
    // over 958 MB 175 us, 171 so; one token behind 517 9.2 and 8.6).
    auto step = [&](auto more) {
      constexpr bool kMore = decltype(more)::value;
      if constexpr (kMore) pages(j0 + 4 * kS, pa, pb);
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      q35_u32x4 kc[2][2];  // 4 bits: a key's 64 codes and two words, 8 keys' 16 codes and word
      u2 vc[8];
      uint32_t kw[2], vw[8];
      if constexpr (k4) {
        wave_lds_sync();  // (the last step's reads)
        store_rows();
        if constexpr (kMore) load_rows(j0 + 4 * kS, pa, pb);
        asm volatile("" ::: "memory");
        wave_lds_sync();
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const char* r = rows_lds + hf * kQ4Half + n * kQ4Row;
          kc[hf][0] = *(const q35_u32x4*)(r + 32 * g);
          kc[hf][1] = *(const q35_u32x4*)(r + 32 * g + 16);
          kw[hf] = *(const uint32_t*)(r + kHd / 2 + 4 * g);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const char* r = rows_lds + (2 + (j >> 2)) * kQ4Half + (4 * g + (j & 3)) * kQ4Row;
          vc[j] = *(const u2*)(r + 8 * n);
          vw[j] = *(const uint16_t*)(r + kHd / 2 + 2 * (n >> 1));
        }
      }
      f4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      // (two sums in turn, the halves' or even and odd dims': a product does not wait for the one before it)
#pragma unroll
      for (int st = 0; st < 8 * kW; ++st) {
        if constexpr (kWide) {
          const q35_u32x4 qv = qs[st * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[0][st][e]), __uint_as_float(qv[e]), sc[e & 1], 0, 0, 0);
        } else if constexpr (k4) {
          q35_u32x4 kv[2];
#pragma unroll
          for (int hf = 0; hf < kH; ++hf) kv[hf] = values8(kc[hf][st >> 2][st & 3], word2(__builtin_amdgcn_perm(kw[hf], kw[hf], st < 4 ? 0x01000100u : 0x03020302u)), nib);
#pragma unroll
          for (int q = 0; q < kQ; ++q) {
            const q35_u32x4 qv = qs[(q * 8 + st) * 64 + lane];
#pragma unroll
            for (int hf = 0; hf < kH; ++hf) sc[hf] = mma<DT>(kv[hf], qv, sc[hf]);
          }
        } else {
#pragma unroll
          for (int q = 0; q < kQ; ++q) {
            const q35_u32x4 qv = qs[(q * 8 + st) * 64 + lane];
#pragma unroll
            for (int hf = 0; hf < kH; ++hf) sc[hf] = mma<DT>(kr[hf][st], qv, sc[hf]);
          }
        }
      }
      if constexpr (kMore && !k4) load_k(j0 + 4 * kS, pa, pb);
      asm volatile("" ::: "memory");
      if constexpr (kWide) sc[0] += sc[1];
      float bm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4 * kH; ++j) {
        const float v = j0 + 16 * (j >> 2) + 4 * g + (j & 3) <= lim ? sc[j >> 2][j & 3] * qscale : -INFINITY;
        sc[j >> 2][j & 3] = v;
        bm = fmaxf(bm, v);
      }
      bm = max_x32(max_x16(bm));
      const float mn = fmaxf(m, bm);
      if (__ballot(mn > m + kSlack)) {
        const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= al;
        m = mn;
      }
      // f16 weights are kept 2^12 times larger (at most 4096, or 2^kSlack times that), so that their halves hold 22 bits down to 2^-26
      const float mr = (m == -INFINITY ? 0.f : m) - (kHalf ? 12.f : 0.f);
      q35_u32x4 pw[kQ];
#pragma unroll
      for (int j = 0; j < 4 * kH; ++j) {
        sc[j >> 2][j & 3] = __builtin_amdgcn_exp2f(sc[j >> 2][j & 3] - mr);
        l += sc[j >> 2][j & 3];
      }
      if constexpr (!kWide) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = sc[j >> 1][2 * (j & 1)], p1 = sc[j >> 1][2 * (j & 1) + 1];
          uint32_t w0, w1, w2 = 0;
          if constexpr (kHalf) split2_near(p0, p1, w0, w1);
          else split3(p0, p1, w0, w1, w2);
          pw[0][j] = w0;
          if constexpr (kQ > 1) pw[1][j] = w1;
          if constexpr (kQ > 2) pw[2][j] = w2;
        }
      }
      if (j0 + kS > end) {  // (uniform) rows behind the sequence's last token may hold anything
#pragma unroll
        for (int j = 0; j < 4 * kH; ++j)
          if (j0 + 16 * (j >> 2) + 4 * g + (j & 3) >= end) {
            if constexpr (k4) {
              vw[j] = 0;
            } else {
#pragma unroll
              for (int w = 0; w < 2 * kW; ++w) vr[j][w] = q35_u32x4{0, 0, 0, 0};
            }
          }
      }
      // 4 bits: tile i: dims 16 (4 g + r) + i in register r
      if constexpr (k4) {
        Word2 w2[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w2[j] = word2(vw[2 * j] | vw[2 * j + 1] << 16);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          q35_u32x4 v[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // byte b of both keys: dims 2 b and 2 b + 1
            const uint32_t t = __builtin_amdgcn_perm(vc[2 * j + 1][b >> 2], vc[2 * j][b >> 2], 0x0c040c00u + (b & 3) * 0x00010001u);
            v[0][j] = low_nibbles(t, w2[j], nib);
            v[1][j] = high_nibbles(t, w2[j], nib);
          }
#pragma unroll
          for (int q = 0; q < kQ; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i) o[2 * b + i] = mma<DT>(v[i], pw[q], o[2 * b + i]);
        }
      } else
      // tile i = w (8 / kW) + e: dims w (128 / kW) + (8 / kW) (4 g + r) + e in register r
#pragma unroll
      for (int w = 0; w < 2 * kW; ++w) {
        if constexpr (kWide) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[j][w][e]), sc[0][j], o[4 * w + e], 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            q35_u32x4 v[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              v[0][j] = __builtin_amdgcn_perm(vr[2 * j + 1][w][e >> 1], vr[2 * j][w][e >> 1], 0x05040100u);
              v[1][j] = __builtin_amdgcn_perm(vr[2 * j + 1][w][e >> 1], vr[2 * j][w][e >> 1], 0x07060302u);
            }
#pragma unroll
            for (int q = 0; q < kQ; ++q)
#pragma unroll
              for (int i = 0; i < 2; ++i) o[8 * w + e + i] = mma<DT>(v[i], pw[q], o[8 * w + e + i]);
          }
        }
      }
      if constexpr (kMore && !k4) load_v(j0 + 4 * kS, pa, pb);
      asm volatile("" ::: "memory");
    };
#pragma unroll 1
    for (; j0 + 4 * kS < j1; j0 += 4 * kS) {
      if constexpr (k4) {
        --left;
        if (left == 3 * quarter) __builtin_amdgcn_s_setprio(2);
        if (left == 2 * quarter) __builtin_amdgcn_s_setprio(1);
        if (left == quarter) __builtin_amdgcn_s_setprio(0);
      }
      step(std::true_type{});
    }
    if (j0 < j1) step(std::false_type{});
    __syncthreads();  // (the queries' operands are done with)
    l = add_x32(add_x16(l));
    if (n < rows) {
      float* dst = os + (wid * kFewRows + n) * kFewLd + (k4 ? 64 * g : (8 / kW) * 4 * g);
      if constexpr (k4) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 16; i += 4) *(f4*)(dst + 16 * r + i) = f4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
      } else
#pragma unroll
      for (int w = 0; w < 2 * kW; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < 8 / kW; e += 4) {
            const int i = w * (8 / kW) + e;
            *(f4*)(dst + w * (128 / kW) + (8 / kW) * r + e) = f4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
          }
      if (g == 0) {
        ms[wid][n] = m;
        ls[wid][n] = l;
      }
    }
    __syncthreads();
    // rows wid, wid + 4, ..: 4 dims per lane
    const bool whole = k0 == 0 && k1 == t.units;
    const int slot = 2 * blockIdx.x + (seg == 0 ? 0 : 1);
#pragma unroll 1
    for (int r = wid; r < rows; r += 4) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) M = fmaxf(M, ms[w][r]);
      float L = 0.f;
      f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = ms[w][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[w][r] - M);
        L += ls[w][r] * f;
        y += *(const f4*)(os + (w * kFewRows + r) * kFewLd + 4 * lane) * f;
      }
      if (whole) {
        const int p2 = t.i * kFewRows + r, tk = div_rep(A, p2), h2 = gk * A.rep + p2 - tk * A.rep;
        const int64_t tr = t.s0 + tk;
        const f4 gv = *(const f4*)(a.qg + tr * a.ld_qg + (int64_t)h2 * 2 * kHd + kHd + 4 * lane);
        const float f = 1.f / L;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = y[e] * f * sigmoid_f(gv[e]);
        *(f4*)(a.out + tr * a.ld_out + (int64_t)h2 * kHd + 4 * lane) = y;
      } else {
        const int64_t pi = (int64_t)slot * A.part_rows[0] + r;
        *(f4*)(A.part_o[0] + pi * kHd + 4 * lane) = y;
        if (lane == 0) {
          A.part_ml[0][2 * pi] = M;
          A.part_ml[0][2 * pi + 1] = L;
          if (k0 == 0) {
            const int p2 = t.i * kFewRows + r, tk = div_rep(A, p2);
            A.cut[(int64_t)(t.s0 + tk) * a.nh + gk * A.rep + p2 - tk * A.rep] = cut_record(slot, r, u, t.units);
          }
        }
      }
    }
    u = k4 && H.whole ? u_end : u + (k1 - k0);
    if (u < u_end && u == t.u0 + (int64_t)t.units * a.nkv) t = uniform(load_tile(&A.tiles[0][++x]));
    __syncthreads();
  }
  if (bad && lane == 0) raise_status(a.status, Q35_STATUS_ARG);
}

// Whether the tiles' w units are read past the 256 MB of the last-level cache: if they are more than it holds, and less
// than an eighth of them is read by another tile too.  (us, through the cache and past it: 33 tokens over 958 MB 206
// and 179; 40 tokens over 800 MB with a tenth shared 144 and 140, a fifth 133 and 140, half 122 and 140; 64 samples
// of 16384 shared tokens 161 and 240; 54 tiles over 229 MB 40 and 53.)
template <int DT>
Q35_DEV bool past_llc(const PlanHead& H, int64_t once) {
  return H.w > (int64_t)(256u << 20) / (kUnit * 2 * kRow<DT> * (int)sizeof(typename Elt<DT>::T)) && 8 * (H.w - once) < H.w;
}

template <int DT>
__global__ __launch_bounds__(kT, 2) void paged_few_kernel(const AttnArgs A) {
  extern __shared__ __align__(16) float os[];
  __shared__ float ms[4][kFewRows], ls[4][kFewRows];
  __shared__ Start sh;
  PlanHead H;
  const int64_t once = *A.once;
  if (!block_start<DT == Q35_Q4>(A, 0, &H, &sh)) return;
  if (past_llc<DT>(H, once)) few_run<DT, true>(A, H, sh, os, ms, ls);
  else few_run<DT, false>(A, H, sh, os, ms, ls);
}

// ------------------------------------------------------------------ many new tokens
// A block takes one tile of up to 128 rows (token, query head of one kv head), 16 per wave, over some
// units.  A unit's keys and values pass LDS, where all eight waves read them.  As above, S^T = K Q^T and
// O^T += V^T P^T (16x16x32 products) keep a row's statistics in its lanes and turn scores into
// operands in place.  16 rows are what leaves two waves a SIMD: a wave's queries (64 or 96 registers)
// and outputs (64) stay in registers that the vector ALU reaches too (with 32 rows per wave, half the
// LDS reads, and one wave per SIMD they did not: 2.5 ms instead of 1.15 for 2048 tokens behind 14336).
// While a unit is multiplied, the next one is on its way into registers; it is then laid out in the
// other LDS buffer, so one barrier per unit is enough.
// LDS: keys [key][32 pieces of 8 dims], piece c at c ^ (key & 15); values [dim][4 pieces of 8 keys], the keys
// in the order of the weights' registers, dim d's row at d ^ (d / 16 % 4), piece c at c ^ (-(d / 4) % 4): a
// 16-byte read serves lanes 0-3, 12-15, 20-23, 24-27 at a time, then 4-11, 16-19, 28-31, and so does the
// upper half; these places lie in different banks each time.
// f16 caches are multiplied with 2 f16 halves of a query or weight, bf16 ones with 3 bf16 parts; f32
// caches as 2 f16 halves with 2 (three products; what is dropped is 2^-24 of a term), under a power of
// two for every 4 keys (a wave's share of the unit) and one for the values.  The values' power comes from the largest
// one that the segment has met, found from 4 keys by each wave: where they differ, the weights make up for it,
// and lose as many bits, so that a unit whose powers differ by more than 2^3 is laid out once more under their
// largest (always under each wave's own, 16384 small weights beside values 2 10^6 times the others were 4 10^-3 off).
// Bound by the matrix cores: 2048 tokens of 8 heads behind 14336 in f32 770-850 us with the card's clock, 300-330
// TFLOP/s of f32 products, 900-990 of f16 ones (a large f16 product of the library: 1112); the whole call 806 us, over
// an f16 cache (two products instead of three) 500, over bf16 (three) 617.
constexpr int kMT = 512;       // threads
constexpr int kRowsW = 16;     // rows of a wave
constexpr int kPlane = 16384;  // bytes of a unit's keys (or values) of one part
template <int DT>
constexpr int many_lds() { return 2 * 2 * kPlane * (DT == Q35_F32 ? 2 : 1); }

// m = max(m, |x|, |y|) of f32 bits (fmaxf quiets its arguments first, an instruction each)
Q35_DEV void max3_abs(float& m, uint32_t x, uint32_t y) { asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(m) : "v"(x), "v"(y)); }
// larger of each 16-bit half
Q35_DEV uint32_t pk_max(uint32_t x, uint32_t y) {
  typedef uint16_t us2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, y)));
}
// f y (f a power of two, y as f32 bits) as f16 halves hi + lo, to nearest: v_fma_mixlo / mixhi multiply in f32, add
// an f16 and round to f16 in one instruction, so a value takes two
Q35_DEV void split2_scaled(uint32_t y0, uint32_t y1, float f, uint32_t& hi, uint32_t& lo) {
  uint32_t h, l;
  asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(y0), "v"(f));
  asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(y1), "v"(f));
  asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(y0), "v"(f), "v"(h));
  asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y1), "v"(f), "v"(h));
  hi = h;
  lo = l;
}

template <int DT>
__global__ __launch_bounds__(kMT) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_many_kernel(const AttnArgs A) {
  typedef typename Elt<DT>::T E;
  constexpr bool kWide = DT == Q35_F32, k4 = DT == Q35_Q4;
  constexpr int kQ = DT == Q35_BF16 ? 3 : 2;  // parts of a query or weight
  constexpr int kKV = kWide ? 2 : 1;          // parts of a key or value
  // how far (log2) a score may pass the running maximum before the sums are rescaled: f16 weights
  // are kept 2^12 times larger and must stay below 2^16
  constexpr float kSlack = DT == Q35_BF16 ? 8.f : 3.f;
  constexpr float kUneven = 0.125f;  // (the largest of 4 x 256 values of one distribution differ by less)
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const PagedAttn& a = A.c;
  extern __shared__ __align__(16) char lds[];  // [2 buffers][keys, values][part]
  __shared__ float scl[2][2][8];               // [buffer][keys, values][group of 4 keys]
  __shared__ Start sh;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4, n32 = lane & 31, hf = lane >> 5;
  PlanHead H;
  if (!block_start<false>(A, 1, &H, &sh)) return;
  const int64_t u_begin = block_u0(H, blockIdx.x);
  int64_t u = u_begin;
  const int64_t u_end = block_u0(H, blockIdx.x + 1);
  Tile t = uniform(load_tile(&sh.t));
  int x = sh.x;
  const float sl2 = a.scale * 1.44269504088896341f;
  const Nibbles nib = nibbles();
  bool bad = false;
  for (int seg = 0; u < u_end; ++seg) {
    int gk = 0;
    int64_t off = u - t.u0;
    for (; off >= t.units; off -= t.units) ++gk;
    const int k0 = (int)off, k1 = (int)min((int64_t)t.units, k0 + (u_end - u));
    const int tok0 = t.i * A.tok_many, rows = min(A.tok_many, t.n - tok0) * A.rep;
    const int r = min(wid * kRowsW + n, rows - 1);  // the lane's row (past the last one: repeated, not written)
    const int tok = tok0 + div_rep(A, r), h = gk * A.rep + r - (tok - tok0) * A.rep;
    const int lim = t.p0 + tok;
    const bool wave_on = wid * kRowsW < rows;
    // the first and the last token that a row of the wave sees
    const int lim0 = t.p0 + tok0 + div_rep(A, min(wid * kRowsW, rows - 1));
    const int lim1 = t.p0 + tok0 + div_rep(A, min(wid * kRowsW + kRowsW - 1, rows - 1));
    const int end = t.p0 + min(tok0 + A.tok_many, t.n);  // no row of the tile sees tokens from here on
    const int32_t* row = a.table + (int64_t)t.b * a.ld_table;
    const E* base = static_cast<const E*>(a.P.data) + (int64_t)a.layer * a.P.n_pages * page_elts<DT>(a) + (int64_t)gk * a.P.page * kRow<DT>;
    // staging registers: keys 4 wid + 2 i + hf, dims 8 n32 ..; values: keys 4 wid + i, dims 4 lane ..
    typedef typename std::conditional<k4, uint32_t, q35_u32x4>::type KW;
    KW kr[2][kKV];
    typedef typename std::conditional<kWide, q35_u32x4, typename std::conditional<k4, uint32_t, u2>::type>::type VW;
    VW vr[4];
    uint32_t kwd[2] = {}, vwd[4] = {};  // 4 bits: their words
    auto unit_page = [&](int k) {  // of the wave's 4 keys
      const int j0 = k * kUnit + 4 * wid;
      return page_of(A, row, j0 < end ? j0 : k * kUnit, &bad);
    };
    auto load_unit = [&](int k, int pg) {
      const int j0 = k * kUnit + 4 * wid;
      const E* p = base + (int64_t)pg * page_elts<DT>(a) + (int64_t)(j0 & (a.P.page - 1)) * kRow<DT>;
      if constexpr (k4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const E* r = p + (2 * i + hf) * kRow<DT>;
          kr[i][0] = *(const Q35_GLOBAL uint32_t*)(r + 4 * n32);
          kwd[i] = *(const Q35_GLOBAL uint16_t*)(r + kHd / 2 + 2 * (n32 >> 2));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const E* r = p + plane_elts<DT>(a) + i * kRow<DT>;
          vr[i] = *(const Q35_GLOBAL uint16_t*)(r + 2 * lane);
          vwd[i] = *(const Q35_GLOBAL uint16_t*)(r + kHd / 2 + 2 * (lane >> 3));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int w = 0; w < kKV; ++w) kr[i][w] = *((const Q35_GLOBAL q35_u32x4*)(p + (2 * i + hf) * kHd + 8 * n32) + w);
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[i] = *(const Q35_GLOBAL VW*)(p + plane_elts<DT>(a) + i * kHd + 4 * lane);
      }
    };
    float vinv = 0.f;  // f32 caches: the power of two that brings the largest value so far to 2^14, its inverse
    auto store_unit = [&](int k, int buf) {
      if (k * kUnit + kUnit > end) {  // (uniform) rows behind the last token may hold anything
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (k * kUnit + 4 * wid + 2 * i + hf >= end) {
            kwd[i] = 0;
#pragma unroll
            for (int w = 0; w < kKV; ++w) kr[i][w] = KW(0);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k * kUnit + 4 * wid + i >= end) {
            vr[i] = VW(0);
            vwd[i] = 0;
          }
      }
      char* kb = lds + buf * 2 * kKV * kPlane;
      char* vb = kb + kKV * kPlane;
      float fk = 1.f, fv = 1.f;
      if constexpr (kWide) {
        // the largest |key| and |value| of the wave's 4 rows, as the upper halves of their bits, in one word
        float mk = 0.f, mv = 0.f, ik, iv;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            max3_abs(mk, kr[i >> 1][i & 1][e], kr[i >> 1][i & 1][e + 1]);
            max3_abs(mv, vr[i][e], vr[i][e + 1]);
          }
        uint32_t m2 = __builtin_amdgcn_perm(__float_as_uint(mv), __float_as_uint(mk), 0x07060302u);
        m2 = pk_max(m2, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m2, 0x128, 0xf, 0xf, false));
        m2 = pk_max(m2, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m2, 0x124, 0xf, 0xf, false));
        m2 = pk_max(m2, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m2, 0x122, 0xf, 0xf, false));
        m2 = pk_max(m2, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m2, 0x121, 0xf, 0xf, false));
        const auto r16 = __builtin_amdgcn_permlane16_swap(m2, m2, false, false);
        m2 = pk_max(r16[0], r16[1]);
        const auto r32 = __builtin_amdgcn_permlane32_swap(m2, m2, false, false);
        m2 = pk_max(r32[0], r32[1]);
        split_scale(__uint_as_float(m2 << 16), fk, ik);  // (the exponent is all that counts)
        split_scale(__uint_as_float(m2 & 0xffff0000u), fv, iv);
        // (2^-100 at least: 2^12 over it stays finite; zeros ask for nothing)
        iv = fmaxf(fmaxf(iv, 7.888609e-31f), vinv);
        fv = __uint_as_float((254u << 23) - __float_as_uint(iv));
        if (m2 >> 16 == 0) iv = 0.f;
        if (lane == 0) {
          scl[buf][0][wid] = ik;
          scl[buf][1][wid] = iv;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = 4 * wid + 2 * i + hf;
        char* dst = kb + key * 512 + (n32 ^ (key & 15)) * 16;
        if constexpr (kWide) {
          q35_u32x4 hi, lo;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1;
            split2_scaled(kr[i][j >> 1][2 * (j & 1)], kr[i][j >> 1][2 * (j & 1) + 1], fk, a0, a1);
            hi[j] = a0;
            lo[j] = a1;
          }
          *(q35_u32x4*)dst = hi;
          *(q35_u32x4*)(dst + kPlane) = lo;
        } else if constexpr (k4) {
          *(q35_u32x4*)dst = values8(kr[i][0], word2(kwd[i] * 0x00010001u), nib);
        } else {
          *(q35_u32x4*)dst = kr[i][0];
        }
      }
      // keys 4 wid .. of dim d: piece wid % 4 (the keys of the weights' lane group), half wid / 4
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        char* dst = vb + (4 * lane + (e ^ ((lane >> 2) & 3))) * 64 + (((wid ^ -lane) & 3) * 16) + (wid >> 2) * 8;
        if constexpr (kWide) {
          uint32_t a0, a1, b0, b1;
          split2_scaled(vr[0][e], vr[1][e], fv, a0, a1);
          split2_scaled(vr[2][e], vr[3][e], fv, b0, b1);
          *(u2*)dst = u2{a0, b0};
          *(u2*)(dst + kPlane) = u2{a1, b1};
        } else if constexpr (k4) {
          const uint32_t c0 = (vr[0] | vr[1] << 16) >> (e & 2) * 4, c1 = (vr[2] | vr[3] << 16) >> (e & 2) * 4;
          const Word2 w0 = word2(vwd[0] | vwd[1] << 16), w1 = word2(vwd[2] | vwd[3] << 16);
          *(u2*)dst = e & 1 ? u2{high_nibbles(c0, w0, nib), high_nibbles(c1, w1, nib)} : u2{low_nibbles(c0, w0, nib), low_nibbles(c1, w1, nib)};
        } else {
          const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
          *(u2*)dst = u2{__builtin_amdgcn_perm(vr[1][e >> 1], vr[0][e >> 1], sel), __builtin_amdgcn_perm(vr[3][e >> 1], vr[2][e >> 1], sel)};
        }
      }
    };
    // The blocks' ranges begin anywhere in their tiles.  The units of a range may come in any order, so a block
    // begins where its unit's number is that of its own steps so far, modulo the units of a block, and goes
    // round: all blocks then look at the same few places of the context at about the same time, and
    // find in the L2 what another has read (2048 tokens behind 14336: 3.5 -> 1.75 GB from behind the L2s).
    const int round = (int)min(H.q, (int64_t)INT32_MAX);
    int ks = k0 + (int)(((u - u_begin - k0) % round + round) % round);
    if (ks >= k1) ks = k0;
    int kn = ks + 1 < k1 ? ks + 1 : k0;  // the next unit
    int pg = unit_page(kn);              // and its page, asked for a unit ahead
    load_unit(ks, unit_page(ks));
    // queries: column n, dims 32 st + 8 g ..
    q35_u32x4 qb[kQ][8];
    float qscale = sl2;
    {
      const int64_t qi = (int64_t)(t.s0 + tok) * a.nh + h;
      float fq = 1.f;
      if constexpr (DT != Q35_BF16) {
        float inv;
        split_scale(A.qmax[qi], fq, inv);
        qscale = sl2 * inv;
      }
#pragma unroll
      for (int st = 0; st < 8; ++st) {
        const float* qp = A.q + qi * kHd + 32 * st + 8 * g;
        const f4 v0 = *(const Q35_GLOBAL f4*)qp, v1 = *(const Q35_GLOBAL f4*)(qp + 4);
        const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p0, p1, p2 = 0;
          if constexpr (k4) split2_near(v[j] * fq, v[j + 4] * fq, p0, p1);  // (values8's order)
          else if constexpr (kQ == 2) split2_near(v[2 * j] * fq, v[2 * j + 1] * fq, p0, p1);
          else split3(v[2 * j], v[2 * j + 1], p0, p1, p2);
          qb[0][st][j] = p0;
          qb[1][st][j] = p1;
          if constexpr (kQ == 3) qb[2][st][j] = p2;
        }
      }
    }
    f4 o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    float ov = DT == Q35_BF16 ? 1.f : 4096.f;  // o is kept this much larger (f32 caches: 2^12 over the values' powers of two)
    // reads: key n (+ 16), pieces 4 st + g; dim 16 dt + n, piece g
    int ka_off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ka_off[i] = n * 512 + ((4 * i + g) ^ n) * 16;
    const int va_off = n * 64 + ((g ^ -(n >> 2)) & 3) * 16;
    int k = ks;
    for (int i = 0, turn = 0; i < k1 - k0; ++turn) {
      const int buf = turn & 1;
      store_unit(k, buf);
      const int j0 = k * kUnit;
      k = kn;
      if (i + 1 < k1 - k0) load_unit(k, pg);
      kn = k + 1 < k1 ? k + 1 : k0;
      pg = unit_page(kn);
      __syncthreads();
      const bool on = wave_on && j0 <= lim1;  // (uniform in the wave; the barriers are passed by all)
      float own = 0.f;
      if constexpr (kWide) own = scl[buf][1][lane & 7];
      const char* kb = lds + buf * 2 * kKV * kPlane;
      const char* vb = kb + kKV * kPlane;
      f4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if (__builtin_expect(on, 1)) {
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          const char* src = kb + ka_off[st & 3] + (st >> 2) * 256;
          q35_u32x4 ka[2][kKV];
#pragma unroll
          for (int w = 0; w < kKV; ++w)
#pragma unroll
            for (int tl = 0; tl < 2; ++tl) ka[tl][w] = *(const q35_u32x4*)(src + tl * 16 * 512 + w * kPlane);
          // (the two tiles in turn: a product does not wait for the one before it)
#pragma unroll
          for (int q = 0; q < kQ; ++q)
#pragma unroll
            for (int tl = 0; tl < 2; ++tl) sc[tl] = mma<DT>(ka[tl][0], qb[q][st], sc[tl]);
          if constexpr (kWide) {
#pragma unroll
            for (int tl = 0; tl < 2; ++tl) sc[tl] = mma<DT>(ka[tl][1], qb[0][st], sc[tl]);
          }
        }
        // operands are read kAhead steps before their products
        constexpr int kAhead = kWide ? 1 : 2;
        constexpr int kKr = 2 * kKV, kKm = 2 * (kWide ? 3 : kQ);  // reads and products of a step
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead * kKr, 0);
#pragma unroll
        for (int st = 0; st < 8 - kAhead; ++st) {
          __builtin_amdgcn_sched_group_barrier(0x008, kKm / 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, kKr / 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, kKm / 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, kKr / 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kAhead * kKm, 0);
      }
      if constexpr (kWide) {
        // the largest of the unit's powers of two; where one is far below it, the unit is laid out again (all waves
        // see the same numbers; then none is: at most once a unit).  Looked for behind the first products, and
        // marked as rare, for the schedule's sake: 830 us for 2048 tokens behind 14336, 847 before them, 821 never.
        float top = fmaxf(own, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(own), 0xB1, 0xf, 0xf, false)));
        top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0x4E, 0xf, 0xf, false)));
        top = fmaxf(top, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(top), 0x141, 0xf, 0xf, false)));
        vinv = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(fmaxf(fmaxf(top, 7.888609e-31f), vinv))));
        if (__builtin_expect(__ballot(own > 0.f && own < vinv * kUneven) != 0, 0)) {
          kn = k;
          pg = unit_page(kn);
          k = j0 / kUnit;
          load_unit(k, unit_page(k));
          continue;
        }
      }
      ++i;
      if (!on) continue;
      float fk[2] = {qscale, qscale}, fp[2] = {4096.f, 4096.f};
      float vscale = ov;
      if constexpr (kWide) {
        vscale = 4096.f * __uint_as_float((254u << 23) - __float_as_uint(vinv));  // the outputs': 2^12 / vinv
#pragma unroll
        for (int tl = 0; tl < 2; ++tl) {
          fk[tl] = scl[buf][0][4 * tl + g] * qscale;
          fp[tl] = scl[buf][1][4 * tl + g] * vscale;  // 2^12 at most
        }
      }
      float bm = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = sc[e >> 2][e & 3] * fk[e >> 2];
        if (j0 + kUnit - 1 > lim0) v = j0 + 16 * (e >> 2) + 4 * g + (e & 3) <= lim ? v : -INFINITY;
        sc[e >> 2][e & 3] = v;
        bm = fmaxf(bm, v);
      }
      bm = max_x32(max_x16(bm));
      if (__ballot(bm > m + kSlack || (m == -INFINITY && bm > m)) || (kWide && vscale != ov)) {
        const float mn = fmaxf(m, bm);
        float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
        m = mn;
        if constexpr (kWide) al *= vscale / ov;
        ov = vscale;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= al;
      }
      const float mr = m == -INFINITY ? 0.f : m;
      q35_u32x4 pw[kQ];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 2 * j;
        float p0 = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - mr), p1 = __builtin_amdgcn_exp2f(sc[e >> 2][(e & 3) + 1] - mr);
        l += p0 + p1;
        if constexpr (DT != Q35_BF16) {
          p0 *= fp[e >> 2];
          p1 *= fp[e >> 2];
        }
        uint32_t w0, w1, w2 = 0;
        if constexpr (kQ == 2) split2_near(p0, p1, w0, w1);
        else split3(p0, p1, w0, w1, w2);
        pw[0][j] = w0;
        pw[1][j] = w1;
        if constexpr (kQ == 3) pw[2][j] = w2;
      }
#pragma unroll
      for (int dt = 0; dt < 16; dt += 2) {
        q35_u32x4 va[2][kKV];
#pragma unroll
        for (int w = 0; w < kKV; ++w)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            va[i][w] = *(const q35_u32x4*)(vb + (va_off ^ (((dt + i) & 3) * 64)) + (dt + i) * 1024 + w * kPlane);
#pragma unroll
        for (int q = 0; q < kQ; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) o[dt + i] = mma<DT>(va[i][0], pw[q], o[dt + i]);
        if constexpr (kWide) {
#pragma unroll
          for (int i = 0; i < 2; ++i) o[dt + i] = mma<DT>(va[i][1], pw[0], o[dt + i]);
        }
      }
      constexpr int kVm = 2 * (kWide ? 3 : kQ), kVr = 2 * kKV, kAheadV = kWide ? 1 : 2;  // of two dims' tiles
      __builtin_amdgcn_sched_group_barrier(0x100, kAheadV * kVr, 0);
#pragma unroll
      for (int dt = 0; dt < 8 - kAheadV; ++dt) {
        __builtin_amdgcn_sched_group_barrier(0x008, kVm / 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kVr / 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, kVm / 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kVr / 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kAheadV * kVm, 0);
    }
    // register e of o[dt] is dim 16 dt + 4 g + e
    l = add_x32(add_x16(l));
    const bool whole = k0 == 0 && k1 == t.units;
    if (wid * kRowsW + n < rows) {
      const float f = (whole ? 1.f / l : 1.f) / ov;
      const int64_t tr = t.s0 + tok;
      const float* gate = a.qg + tr * a.ld_qg + (int64_t)h * 2 * kHd + kHd;
      const int64_t pi = (int64_t)(2 * blockIdx.x + (seg == 0 ? 0 : 1)) * A.part_rows[1] + r;
      float* dst = whole ? a.out + tr * a.ld_out + (int64_t)h * kHd : A.part_o[1] + pi * kHd;
      // (the empty asm keeps these addresses from being formed before the loop, where they cost its operands
      // their registers)
      int ge = 4 * g;
      asm volatile("" : "+v"(ge));
      gate += ge;
      dst += ge;
      if (whole) {
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
          const f4 gv = *(const f4*)(gate + 16 * dt);
          f4 y = o[dt] * f;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] *= sigmoid_f(gv[e]);
          *(f4*)(dst + 16 * dt) = y;
        }
      } else {
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) *(f4*)(dst + 16 * dt) = o[dt] * f;
      }
      if (!whole && g == 0) {
        A.part_ml[1][2 * pi] = m;
        A.part_ml[1][2 * pi + 1] = l;
        if (k0 == 0)
          A.cut[tr * a.nh + h] = cut_record(2 * blockIdx.x + (seg == 0 ? 0 : 1), -1 - r, u, t.units);
      }
    }
    u += k1 - k0;
    if (u < u_end && u == t.u0 + (int64_t)t.units * a.nkv) t = uniform(load_tile(&A.tiles[1][++x]));
    __syncthreads();  // (the buffers are the next segment's)
  }
  if (bad && lane == 0) raise_status(a.status, Q35_STATUS_ARG);
}

// Joins the parts of a row's tile, if the plan cut it: kJW waves per (row, query head), each taking every
// kJW-th part, eight of them in flight.  Bound by round trips (one token 4.4 us) or the parts' stream (8720 rows of
// mixed batch, most of them of 5 parts, 11.8).
template <int kJW>
__global__ __launch_bounds__(kT) void paged_join_kernel(const AttnArgs A) {
  const PagedAttn& a = A.c;
  __shared__ __align__(16) float ys[kJW > 1 ? kT / 64 : 1][kHd];
  __shared__ float ls[kT / 64];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), jw = wid % kJW;
  const int64_t item = (int64_t)blockIdx.x * (kT / 64 / kJW) + wid / kJW;
  const int64_t t = item / a.nh;
  const int h = (int)(item % a.nh);
  if (t >= a.T) return;
  // (asked for together: the record, the plan's heads and the gate, then the statistics and the first parts)
  const int4 c = A.cut[t * a.nh + h];
  const PlanHead head[2] = {A.head[0], A.head[1]};
  if (c.x == 0) return;  // (kJW > 1: the block's waves share their item, and leave together)
  const f4 gv = *(const f4*)(a.qg + t * a.ld_qg + (int64_t)h * 2 * kHd + kHd + 4 * lane);
  const int kind = c.y < 0 ? 1 : 0, r = kind ? -1 - c.y : c.y, g0 = (c.x - 1) >> 1;
  const int np = unit_block(kind ? head[1] : head[0], (int64_t)c.w << 32 | (uint32_t)c.z) - g0 + 1;
  auto slot = [&](int q) { return (int64_t)(q == 0 ? c.x - 1 : 2 * (g0 + q)) * A.part_rows[kind] + r; };
  const float* ml = A.part_ml[kind];
  f4 v[8];
  float w[8], lw[8];
  auto load = [&](int q0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t o = slot(min(q0 + e * kJW, np - 1));
      v[e] = *(const Q35_GLOBAL f4*)(A.part_o[kind] + o * kHd + 4 * lane);
      w[e] = ml[2 * o];
      lw[e] = ml[2 * o + 1];
    }
  };
  load(jw);
  float M = -INFINITY;
  for (int q = lane; q < np; q += 64) M = fmaxf(M, ml[2 * slot(q)]);
#pragma unroll
  for (int e = 32; e > 0; e >>= 1) M = fmaxf(M, __shfl_xor(M, e, 64));
  float L = 0.f;
  f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int q0 = jw; q0 < np; q0 += 8 * kJW) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // (a part none of whose tokens the row sees has the maximum -inf and zeros)
      const float f = q0 + e * kJW < np ? __builtin_amdgcn_exp2f(w[e] - M) : 0.f;
      L += lw[e] * f;
      y += v[e] * f;
    }
    if (q0 + 8 * kJW < np) load(q0 + 8 * kJW);
  }
  if constexpr (kJW > 1) {
    *(f4*)&ys[wid][4 * lane] = y;
    if (lane == 0) ls[wid] = L;
    __syncthreads();
    if (wid != 0) return;
#pragma unroll
    for (int w = 1; w < kJW; ++w) {
      y += *(const f4*)&ys[w][4 * lane];
      L += ls[w];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = y[e] / L * sigmoid_f(gv[e]);
  *(f4*)(a.out + t * a.ld_out + (int64_t)h * kHd + 4 * lane) = y;
}

struct PagedLayout {
  int32_t max_tiles[2], max_blocks[2], part_rows[2], few_most;
  size_t head, tile0, q, qmax, cut, tiles[2], ml[2], o[2];  // byte sizes
  size_t bytes;
};
// What all tiles of T rows, as "few", may go over if all are one sequence's: tiles, kv heads, tokens, bytes of a value.
constexpr int64_t kReread = 300000, kReread4 = 350000;
// ctx_bytes: tokens that a sequence can have, times the bytes of a value; INT64_MAX for the workspace of any call.
PagedLayout paged_layout(int nh, int nkv, int T, int B, int64_t ctx_bytes, bool k4) {
  PagedLayout L;
  const int rep = nh / nkv, tok_many = kManyRows / rep;
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  // A sequence of two tiles of "few" rows, or of one token, is "few": 5 drafted tokens of 4 heads (20 rows) behind
  // 100 take 9.4 us there and 17.8 as a chunk.  16 tokens (4 tiles) take 20 us behind 200 and 98 behind 30000 in
  // f32, 32 and 47 as a chunk: every tile reads the context again.
  // Which kinds there are is the device's knowledge; what a call cannot or need not have gets no launch (an
  // empty one takes 1.7 us, 3 where the host is behind).  If no sequence is empty, the longest has T - B + 1 tokens
  // at most: where that is "few", all are (were all "few" up to two tokens per sequence, 63 of one token behind
  // 2000 and one of 64 behind 30000 would take 207 us, 133 so).  But a batch of fixed slots may be one chunk and
  // empty ones, so that holds only while the chunk's tiles could go over the longest context that the table
  // and the rotary rows allow as cheaply as a chunk does (kReread; both ways, us: 16 tokens behind 16000 in bf16 37
  // and 37, in f32 54 and 40; 64 behind 2000 28 and 37, 36 and 40; 256 behind 16000 272 and 112, 572 and 134).
  // Over 4 bits, where one chunk of all rows would cost no more in tiles, any batch goes so that has as many tiles as blocks at
  // most (both ways, us: 16 tokens behind 60000 in a padded batch 48 and 53, 64 behind 16000 46 and 54, 256 behind 5000 60 and 60,
  // 500 behind 2000 63 and 63, behind 2600 73 and 69; 48 behind 16000 beside 12 single ones 49 and 70; 10 prompts of 100 31 and
  // 64, 20 of 200, 1000 tiles, 148 and 102; one of 64 16 and 45, of 500 35 and 63, 500 behind 1500 57 and 57).  What counts is what
  // the table and the rotary rows could hold: under ones for 4096 tokens 10 prompts of 100 take 64, for 32768 one of 64 takes 45.
  // Else, one sequence: its rows decide, if all rows are its.
  L.few_most = std::max(1, 2 * kFewRows / rep);
  const int64_t tiles = ((int64_t)T * rep + kFewRows - 1) / kFewRows * nkv;
  const bool cheap = ctx_bytes <= (k4 ? kReread4 : kReread) / tiles;
  const bool few_only = T <= L.few_most || (cheap && (k4 ? tiles <= 2 * device_cus() : T - B + 1 <= L.few_most));
  const bool many_only = !few_only && B == 1;
  if (few_only) L.few_most = INT_MAX;
  if (many_only) L.few_most = 0;
  const int seqs = std::min(B, T);
  L.max_tiles[0] = many_only ? 0 : (int)(((int64_t)T * rep + kFewRows - 1) / kFewRows + seqs);
  L.max_tiles[1] = few_only ? 0 : T / tok_many + seqs;
  const int cus = device_cus();
  L.max_blocks[0] = many_only ? 0 : 2 * cus;
  L.max_blocks[1] = few_only ? 0 : cus;
  L.part_rows[0] = (int)std::min<int64_t>(kFewRows, (int64_t)T * rep);
  L.part_rows[1] = (int)std::min<int64_t>(kManyRows, (int64_t)T * rep);
  L.head = up(2 * sizeof(PlanHead) + sizeof(int64_t));
  L.tile0 = up((size_t)2 * B * 4);
  L.q = up((size_t)T * nh * kHd * 4);
  L.qmax = up((size_t)T * nh * 4);
  L.cut = up((size_t)T * nh * sizeof(int4));
  L.bytes = L.head + L.tile0 + L.q + L.qmax + L.cut;
  for (int k = 0; k < 2; ++k) {
    const size_t rows = (size_t)2 * L.max_blocks[k] * L.part_rows[k];
    L.tiles[k] = up((size_t)L.max_tiles[k] * sizeof(Tile));
    L.ml[k] = up(rows * 8);
    L.o[k] = up(rows * kHd * 4);
    L.bytes += L.tiles[k] + L.ml[k] + L.o[k];
  }
  return L;
}

template <int DT>
int launch(const PagedAttn& a, hipStream_t st) {
  const int64_t ctx = std::min<int64_t>((int64_t)a.ld_table * a.P.page, a.rope_rows);
  const PagedLayout L = paged_layout(a.nh, a.nkv, a.T, a.B, ctx * row_bytes(a.P) / kHd, DT == Q35_Q4);
  AttnArgs A;
  A.c = a;
  A.page_shift = __builtin_ctz((unsigned)a.P.page);
  A.rep = a.nh / a.nkv;
  A.rep_inv = A.rep > 1 ? (uint32_t)(0x100000000ull / (uint32_t)A.rep) + 1u : 0u;
  A.tok_many = kManyRows / A.rep;
  A.few_most = L.few_most;
  char* p = static_cast<char*>(a.ws);
  A.head = reinterpret_cast<PlanHead*>(p);
  A.once = reinterpret_cast<int64_t*>(A.head + 2);
  p += L.head;
  A.tile0 = reinterpret_cast<int32_t*>(p);
  p += L.tile0;
  A.q = reinterpret_cast<float*>(p);
  p += L.q;
  A.qmax = reinterpret_cast<float*>(p);
  p += L.qmax;
  A.cut = reinterpret_cast<int4*>(p);
  p += L.cut;
  for (int k = 0; k < 2; ++k) {
    A.max_tiles[k] = L.max_tiles[k];
    A.max_blocks[k] = L.max_blocks[k];
    A.part_rows[k] = L.part_rows[k];
    A.tiles[k] = reinterpret_cast<Tile*>(p);
    p += L.tiles[k];
    A.part_ml[k] = reinterpret_cast<float*>(p);
    p += L.ml[k];
    A.part_o[k] = reinterpret_cast<float*>(p);
    p += L.o[k];
  }
  const int64_t ka = (int64_t)a.T * (a.nkv + a.nh), qa = (int64_t)a.T * a.nh;
  hipLaunchKernelGGL(paged_append_kernel<DT>, dim3((uint32_t)((ka + 3) / 4 + 2)), dim3(kT), 0, st, A);
  Q35_HIP_TRY(hipGetLastError());
  if (A.max_blocks[0] > 0) {
    allow_lds<paged_few_kernel<DT>>(kFewLds);
    hipLaunchKernelGGL(paged_few_kernel<DT>, dim3(A.max_blocks[0]), dim3(kT), kFewLds, st, A);
    Q35_HIP_TRY(hipGetLastError());
  }
  if (A.max_blocks[1] > 0) {
    allow_lds<paged_many_kernel<DT>>(many_lds<DT>());
    hipLaunchKernelGGL(paged_many_kernel<DT>, dim3(A.max_blocks[1]), dim3(kMT), many_lds<DT>(), st, A);
    Q35_HIP_TRY(hipGetLastError());
  }
  // few rows: their parts are many, or the chip is empty
  if (qa <= 4096) hipLaunchKernelGGL(paged_join_kernel<4>, dim3((uint32_t)qa), dim3(kT), 0, st, A);
  else hipLaunchKernelGGL(paged_join_kernel<1>, dim3((uint32_t)((qa + 3) / 4)), dim3(kT), 0, st, A);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

}  // namespace

size_t paged_attn_ws_bytes(int nh, int nkv, int T, int B) {
  // (for any type and context: one sequence may be a chunk or few tokens)
  return std::max(paged_layout(nh, nkv, T, B, INT64_MAX, false).bytes, paged_layout(nh, nkv, T, B, 0, true).bytes);
}

int paged_attn_launch(const PagedAttn& a, hipStream_t st) {
  switch (a.P.dtype) {
    case Q35_F32: return launch<Q35_F32>(a, st);
    case Q35_F16: return launch<Q35_F16>(a, st);
    case Q35_Q4: return launch<Q35_Q4>(a, st);
    default: return launch<Q35_BF16>(a, st);
  }
}

}  // namespace q35

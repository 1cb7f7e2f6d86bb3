// The next beams of groups of beams: of all continuations (beam w, token v) of a group the k with the highest
// score[w] + x[w][v] - ln sum e^x[w].
//
// In a row the sum of the logarithm is the same for all tokens, so a row's best continuations are its highest
// logits.  One pass over the logits (blocks (row, part)) keeps each part's k highest and its maximum m and sum
// S of e^(x - m); a block per group then forms the rows' logarithms and chooses among the parts' lists.  Rows that
// have ended or whose beam is dead are not read.
// Continuations of different beams lie close together, and which ones are chosen should hang on as few roundings as it
// can: sums over lanes and parts, logarithms and scores are f64.  f32 are the exponentials and the sums of a lane's 16 of a chunk.
// With u = 2^-24 a term at distance d below its lane's highest so far is off by u (2 + 2.23 d), the sum of 16 by 5 u, and each rise of a
// running maximum by e by u (2 + e): ln sum e^x by u (7 + 2 n + 2.23 D) at most, n the rises above a term and D its distance from the
// row's highest logit, both weighted by the terms' shares.  Measured: 1.5 to 3 10^-8 rms over rows of normal (sigma 0.5 .. 4)
// and of Zipf's logits, 10^-7 at most; up to 2.3 10^-7 where one to three tokens hold the mass (nothing means out there; 7 10^-7
// by the bound) and in rows that rise by less than an exponential's error from chunk to chunk.  Two beams' scores change
// places if they lie within that.
#include "toplist.h"

#include <algorithm>

namespace q35 {

namespace {

constexpr int kT = 256;
constexpr int kNW = kT / 64;
constexpr int kJoinWaves = 16;
constexpr int kBlocks = 4 * 256;  // that rows are cut into
constexpr int kLiveMax = 4096;    // rows among which a block looks for the live ones
constexpr int kMaxLists = 512;    // of a group
constexpr int kListsLane = kMaxLists / 64;
constexpr int kMaxCand = 512;     // that a group's choice ranks by comparing each with each

struct alignas(16) Part {
  double s;
  float m, pad;
};
struct BeamArgs {
  BeamCall c;
  int32_t nsplit;  // parts per row; 0: the device decides, by the number of live rows (split_live)
  int32_t most;    // parts per row at most, and that a row has room for
  int32_t* live;   // live rows
  Part* part;      // [row][most]
  key_t* keys;     // [row][most][k]
};
// Parts of each of n live rows: enough to fill the chip, of one chunk per wave at least.
__host__ __device__ inline int split_live(int n, int most) {
  const int want = n > 0 ? kBlocks / n : 1;
  return want < 1 ? 1 : want < most ? want : most;
}
// The same for the live rows that the device has counted: where a chunk per wave would still fill the chip with more than two
// blocks a CU, two chunks leave half as many lists to join (16 first steps of 8 beams 22.2 -> 20.6 us of a call among others).
Q35_DEV int split_counted(int n, int most) {
  const int ns = split_live(n, most);
  return ns == most && n * most > kBlocks / 2 ? (most + 1) / 2 : ns;
}

// e^d for d <= 0, off by the hardware's 2^-23 at most whatever d
Q35_DEV double exp_near(float d) {
  d = fmaxf(d, -1e4f);
  const float t = d * 1.44269502162933350f;
  const float e = __builtin_fmaf(d, 1.44269502162933350f, -t) + d * 1.92596299112661746e-8f;
  const double p = (double)__builtin_amdgcn_exp2f(t);
  return p + p * (double)(e * 0.693147180559945309f);
}
// ln s, s > 0: the exponent apart, the rest f in [0.7, 1.42) by 2 atanh((f - 1) / (f + 1)), off by 10^-13
Q35_DEV double ln_near(double s) {
  int e;
  double f = frexp(s, &e);
  if (f < 0.70710678118654752) {
    f += f;
    --e;
  }
  const double z = (f - 1.0) / (f + 1.0), z2 = z * z;
  double p = 1.0 / 13.0;
#pragma unroll
  for (int i = 11; i > 0; i -= 2) p = p * z2 + 1.0 / i;
  return (double)e * 0.693147180559945309 + 2.0 * z * p;
}

enum { kDead = 0, kLive = 1, kEnded = 2 };
Q35_DEV int beam_state(const BeamCall& c, int row) {
  if (!(fabsf(c.scores[row]) < INFINITY)) return kDead;
  const int e = c.ended ? c.ended[row] : -1;
  return e < 0 ? kLive : e < c.V ? kEnded : kDead;
}

// 16 bytes at any multiple of 2.  Which lane sums what must hang on a value's index in its row alone, not on the row's
// address: beams with the same logits then have the same sums, and equal scores stay equal.
Q35_DEV uint4 ldg16_any(const void* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  const u4 v = __builtin_nontemporal_load((const Q35_GLOBAL u4*)p);
  return make_uint4(v.x, v.y, v.z, v.w);
}

// Blocks (row, part).  Bound by the stream for many rows (236 live rows of 248320 f32 values 53 us, 4.4 TB/s, the lists' first
// chunks and the blocks' ends beside it; in 16 bits as long, 256 rows 62 and 64 us of a call: the vector work per value), by round trips
// for few (4 rows 8.6 us).
template <int DT>
__global__ __launch_bounds__(kT) void beam_score_kernel(const BeamArgs a) {
  const BeamCall& c = a.c;
  __shared__ key_t lists[kNW][kMaxTop];
  __shared__ key_t buf[kNW][64];
  __shared__ float stage[kNW][kPer][64];
  __shared__ float sm[kNW];
  __shared__ double ss[kNW];
  __shared__ key_t block_last;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int ns = a.nsplit, row_i;
  if (ns > 0) {
    row_i = blockIdx.x / ns;
    if (beam_state(c, row_i) != kLive) return;
  } else {
    // Dead and ended rows leave their blocks to the others (a first step has one live beam of each group, calls, us: 16 of 128 rows
    // of 248320 f16 values 35 in blocks of their own rows, 20.6 so; 100 of 800 of 50257 45 and 25; 250 of 2000 of 32000 57 and 28; 1024 of
    // 4096 84 and 52).  Where all rows live, each block's look at all of them is lost: 256 rows 60.5 and 62.2, 800 46.7 and 48.9, 2000
    // 58 and 66, 4096 85 and 116.
    __shared__ uint16_t live[kLiveMax];
    __shared__ int count[kNW];
    const int M = c.R * c.W;
    int n = 0;
    for (int r0 = 0; r0 < M; r0 += kT) {
      const int r = r0 + tid;
      const bool in = r < M && beam_state(c, r) == kLive;
      const unsigned long long mask = __ballot(in);
      if (lane == 0) count[wid] = __popcll(mask);
      __syncthreads();
      int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
#pragma unroll
      for (int w = 0; w < kNW; ++w) {
        at += w < wid ? count[w] : 0;
        n += count[w];
      }
      if (in) live[at] = (uint16_t)r;
      __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) *a.live = n;
    ns = split_counted(n, a.most);
    if ((int)(blockIdx.x / ns) >= n) return;
    row_i = live[blockIdx.x / ns];
  }
  const int sp = blockIdx.x % ns, len = (c.V + ns - 1) / ns;
  constexpr int kEs = DT == Q35_F32 ? 4 : 2, kVec = 16 / kEs;
  const char* row = static_cast<const char*>(c.x) + (int64_t)row_i * c.ld * kEs;
  const int i0 = min(c.V, sp * len), i1 = min(c.V, i0 + len);  // (a last part may be empty)
  const int top = c.k;
  constexpr int kWords = kPer / kVec;
  constexpr uint32_t kAll = (1u << kPer) - 1u;
  float m = -INFINITY;
  double S = 0.0;
  key_t best = 0, last = 0;
  bool first = true;
  if (tid == 0) block_last = 0;
  __syncthreads();
  for (int64_t f64 = i0 + wid * kChunk; f64 < i1; f64 += kNW * kChunk) {
    float x[kPer];
    uint32_t ok = kAll;
    const int f0 = (int)f64;
    const bool whole = f64 + kChunk <= i1;
    auto index = [&](int e) { return f0 + (e / kVec * 64 + lane) * kVec + e % kVec; };
    if (whole) {
      uint4 v[kWords];
#pragma unroll
      for (int g = 0; g < kWords; ++g) v[g] = ldg16_any(row + (int64_t)f0 * kEs + (g * 64 + lane) * 16);
#pragma unroll
      for (int g = 0; g < kWords; ++g) {
        const uint32_t d[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          x[g * kVec + j] = DT == Q35_F32 ? __uint_as_float(d[j & 3]) : half_of<DT>(d[(j >> 1) & 3], j & 1);
      }
    } else {
      ok = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int f = index(e);
        const float v = value<DT>(row, min(f, i1 - 1));
        const bool in = f < i1;
        x[e] = in ? v : -INFINITY;
        ok |= (in ? 1u : 0u) << e;
      }
    }
    const key_t bl = __hip_atomic_load(&block_last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) mx = fmaxf(mx, x[e]);
    const float mn = fmaxf(m, mx), r = mn == -INFINITY ? 0.f : mn;
    if (__ballot(mn > m && S > 0.0)) S *= exp_near(m - r);
    m = mn;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < kPer; ++e) s[e & 3] += exp_d(x[e] - r);
    S += (double)((s[0] + s[1]) + (s[2] + s[3]));
    list_chunk(x, mx, ok, whole, index, bl, first, best, last, top, stage[wid], buf[wid], &block_last);
  }
  // lanes, then waves
  float M = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  S *= exp_near(m - (M == -INFINITY ? 0.f : M));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) S += __shfl_xor(S, o, 64);
  if (lane == 0) {
    sm[wid] = M;
    ss[wid] = S;
  }
  lists[wid][lane] = best;
  __syncthreads();
  const int64_t slot = (int64_t)row_i * a.most + sp;
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kNW; ++w) M = fmaxf(M, sm[w]);
    const float r = M == -INFINITY ? 0.f : M;
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kNW; ++w) all += ss[w] * exp_near(sm[w] - r);
    a.part[slot] = Part{all, M, 0.f};
  }
  if (lane < top) {
    // the key's place among the block's: its own list's keys before it, and the other lists' larger ones
    int at[kNW] = {};
#pragma unroll 1
    for (int step = 1 << (31 - __clz(top)); step > 0; step >>= 1) {
#pragma unroll
      for (int w = 0; w < kNW; ++w)
        if (at[w] + step <= top && lists[w][at[w] + step - 1] > best) at[w] += step;
    }
    int place = 0;
#pragma unroll
    for (int w = 0; w < kNW; ++w) place += at[w];
    if (best != 0 && place < top) a.keys[slot * top + place] = best;
    // a part with fewer values than `top` leaves the rest of its list empty
    if (wid == 0 && lane >= min(top, i1 - i0)) a.keys[slot * top + lane] = 0;
  }
}

// A continuation: its score's bits in ascending order (0: none), its beam, and its logit and token as a list's key.  Among
// equal scores (which two logits of a beam have where its own score is many times larger) the lower beam is first, then the larger key.
struct Cand {
  unsigned long long hi;
  key_t key;
  uint32_t w;
};
Q35_DEV bool ahead(const Cand& a, const Cand& b) { return a.hi > b.hi || (a.hi == b.hi && (a.w < b.w || (a.w == b.w && a.key > b.key))); }
constexpr uint32_t kNoBeam = ~0u;
Q35_DEV unsigned long long asc64(double c) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, c + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
Q35_DEV double from_asc64(unsigned long long a) { return __builtin_bit_cast(double, a >> 63 ? a & ~(1ull << 63) : ~a); }
Q35_DEV Cand lane_cand(const Cand& c, int lane) {
  return Cand{lane_key(c.hi, lane), lane_key(c.key, lane), (uint32_t)__builtin_amdgcn_readlane((int)c.w, lane)};
}
Q35_DEV unsigned long long lane_before(unsigned long long v) {  // (lane 0: all ones)
  return ((unsigned long long)(uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(v >> 32), 0x138, 0xf, 0xf, false) << 32) |
         (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(uint32_t)v, 0x138, 0xf, 0xf, false);
}
// Puts c (the same in every lane) into the sorted list that the lanes hold; last: its top-th
Q35_DEV void insert_cand(Cand& best, Cand& last, const Cand& c, int top) {
  if (!ahead(c, last)) return;
  const Cand up = {lane_before(best.hi), lane_before(best.key), (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best.w, 0x138, 0xf, 0xf, false)};
  // a place takes the first of what it has and of the second of c and the one before it
  const Cand in = ahead(up, c) ? c : up;
  if (ahead(in, best)) best = in;
  if ((int)(threadIdx.x & 63) >= top) best = Cand{0, 0, kNoBeam};
  last = lane_cand(best, top - 1);
}

// The r-th largest of the wave's N values per lane without its lowest 12 bits; 0 if fewer than r are above 0.  (Two bits a
// step, a score's 12 highest significant bits: each step waits for its counts; 32 steps of one took 3.6 us for 244 lists.)
template <int N>
Q35_DEV uint32_t nth_largest(const uint32_t (&v)[kListsLane], int r) {
  uint32_t t = 0;
#pragma unroll 1
  for (int bit = 30; bit >= 12; bit -= 2) {
    int n[3] = {0, 0, 0};
#pragma unroll
    for (int q = 0; q < N; ++q)
#pragma unroll
      for (int e = 0; e < 3; ++e) n[e] += __popcll(__ballot(v[q] >= (t | (uint32_t)(e + 1) << bit)));
    t |= (uint32_t)((n[0] >= r ? 1 : 0) + (n[1] >= r ? 1 : 0) + (n[2] >= r ? 1 : 0)) << bit;
  }
  return t;
}

// Block per group: the rows' logarithms, then the choice among the parts' lists.
// If r lists have their 2^i-th continuation at or above f, and 2^i r >= k, nothing below f is chosen.  The
// largest such f of all i (of scores as f32, which is monotonic) leaves little more than k continuations; those are
// put into LDS, and each one's place is the number of those ahead of it.  Where many are equal and more are left than LDS
// takes, the waves keep sorted lists instead.
// Bound by round trips (live rows; sums and lists) and short serial steps: 11 us for 32 groups of 8 beams, with sorted
// lists only 14.6; 6.6 for one group of 4.
__global__ __launch_bounds__(kJoinWaves * 64) void beam_join_kernel(const BeamArgs a) {
  const BeamCall& c = a.c;
  __shared__ double off[kMaxBeams];
  __shared__ int state[kMaxBeams];
  __shared__ unsigned long long chi[kMaxCand];
  __shared__ key_t ckey[kMaxCand];
  __shared__ uint32_t cw[kMaxCand];
  __shared__ uint32_t fl;
  __shared__ int nc;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x / 64;
  const int g = blockIdx.x, W = c.W, k = c.k, most = a.most;
  const int64_t row0 = (int64_t)g * W;
  const key_t* keys = a.keys + row0 * most * k;
  if (tid == 0) {
    fl = 1;
    nc = 0;
  }
  const int ns = a.nsplit > 0 ? a.nsplit : split_counted(*a.live, most), nl = W * ns;
  const int levels = 32 - __clz(k), nq = (nl + 63) / 64;
  auto list = [&](int l, int& w, int& sp) {  // the keys of list l
    w = l / ns;
    sp = l - w * ns;
    return keys + ((int64_t)w * most + sp) * k;
  };
  // Asked for together: the thread's list's first keys, the keys of the wave's level (of rows that are not live too:
  // whatever the workspace holds, left aside below), and the sums.
  constexpr int kFirst = 4;
  key_t first[kFirst], level[kListsLane];
  int my_w, my_sp;
  const key_t* my_keys = list(min(tid, nl - 1), my_w, my_sp);
#pragma unroll
  for (int j = 0; j < kFirst; ++j) first[j] = tid < nl && j < k ? my_keys[j] : 0;
  auto ask = [&](int i) {
#pragma unroll
    for (int q = 0; q < kListsLane; ++q) {
      const int l = q * 64 + lane;
      int w, sp;
      level[q] = q < nq && l < nl ? list(l, w, sp)[(1 << i) - 1] : 0;
    }
  };
  if (wid < levels) ask(wid);
#pragma unroll 1
  for (int w = wid; w < W; w += nw) {
    const int row = (int)row0 + w, st = beam_state(c, row);
    const Part* part = a.part + (int64_t)row * most;
    const Part p0 = part[min(lane, ns - 1)];
    double o = c.scores[row];
    if (st == kLive) {
      float m = lane < ns ? p0.m : -INFINITY;
      double S = lane < ns ? p0.s : 0.0;
#pragma unroll 1
      for (int i = lane + 64; i < ns; i += 64) {
        const Part p = part[i];
        const float mn = fmaxf(m, p.m), r = mn == -INFINITY ? 0.f : mn;
        S = S * exp_near(m - r) + p.s * exp_near(p.m - r);
        m = mn;
      }
#pragma unroll 1
      for (int e = 32; e > 0; e >>= 1) {
        const float om = __shfl_xor(m, e, 64), mn = fmaxf(m, om), r = mn == -INFINITY ? 0.f : mn;
        const double oS = __shfl_xor(S, e, 64);
        S = S * exp_near(m - r) + oS * exp_near(om - r);
        m = mn;
      }
      // (NaN or +inf in the row: S is NaN; -inf alone: 0)
      o = S > 0.0 ? o - ((double)m + ln_near(S)) : -INFINITY;
    }
    if (lane == 0) {
      off[w] = o;
      state[w] = st;
      if (c.ended && c.ended[row] >= c.V) raise_status(c.status, Q35_STATUS_ARG);
    }
  }
  __syncthreads();
  // continuation j of part sp of beam w, and its score's f32; 0: none
  auto cand = [&](key_t key, int w, int sp, int j, Cand& x) {
    const int st = state[w];
    double s = -INFINITY;
    if (st == kLive && key != 0) {
      s = off[w] + (double)from_asc((uint32_t)(key >> 32));
    } else if (st == kEnded && sp == 0 && j == 0) {
      s = off[w];
      key = (uint32_t)~c.ended[row0 + w];
    }
    const bool some = s > -INFINITY;
    x = Cand{some ? asc64(s) : 0, key, (uint32_t)w};
    return some ? asc((float)s) : 0u;
  };
#pragma unroll 1
  for (int i = wid; i < levels; i += nw) {
    uint32_t v[kListsLane] = {};
    const int j = (1 << i) - 1;
    if (i != wid) ask(i);
#pragma unroll
    for (int q = 0; q < kListsLane; ++q) {
      const int l = q * 64 + lane;
      if (q < nq && l < nl) {
        const int w = l / ns;
        Cand x;
        v[q] = cand(level[q], w, l - w * ns, j, x);
      }
    }
    const int r = (k + j) >> i;
    const uint32_t f = nq == 1 ? nth_largest<1>(v, r) : nq <= 4 ? nth_largest<4>(v, r) : nth_largest<kListsLane>(v, r);
    if (lane == 0 && f > 1) atomicMax(&fl, f);
  }
  __syncthreads();
  const uint32_t floor32 = fl;
  if (tid < nl) {
#pragma unroll 1
    for (int j = 0; j < k; ++j) {
      const key_t key = first[0];
#pragma unroll
      for (int e = 1; e < kFirst; ++e) first[e - 1] = first[e];
      first[kFirst - 1] = j + kFirst < k ? my_keys[j + kFirst] : 0;
      Cand x;
      if (cand(key, my_w, my_sp, j, x) < floor32) break;  // (lists fall)
      const int at = atomicAdd(&nc, 1);
      if (at < kMaxCand) {
        chi[at] = x.hi;
        ckey[at] = x.key;
        cw[at] = x.w;
      }
    }
  }
  __syncthreads();
  auto put = [&](const Cand& x, int place) {
    const int64_t at = (int64_t)g * k + place;
    c.scores_out[at] = (float)from_asc64(x.hi);
    c.parents[at] = (int32_t)(row0 + x.w);
    c.tokens[at] = key_index(x.key);
  };
  int all = nc;
  if (all <= kMaxCand) {
    for (int t = tid; t < all; t += blockDim.x) {
      const Cand x = {chi[t], ckey[t], cw[t]};
      int place = 0, equal = 0;
      for (int e = 0; e < all; ++e) {
        place += chi[e] > x.hi ? 1 : 0;
        equal += chi[e] == x.hi ? 1 : 0;
      }
      if (equal > 1) {
        for (int e = 0; e < all; ++e) place += chi[e] == x.hi && ahead(Cand{chi[e], ckey[e], cw[e]}, x) ? 1 : 0;
      }
      if (place < k) put(x, place);
    }
  } else {
    // lists by waves: sorted, then joined
    __shared__ Cand sorted[kJoinWaves][kMaxTop];
    Cand best = {0, 0, kNoBeam}, last = best;
#pragma unroll 1
    for (int l0 = wid * 64; l0 < nl; l0 += nw * 64) {
      int w, sp;
      const key_t* held = list(min(l0 + lane, nl - 1), w, sp);
#pragma unroll 1
      for (int j = 0; j < k; ++j) {
        Cand x = {0, 0, kNoBeam};
        const uint32_t a32 = l0 + lane < nl ? cand(held[j], w, sp, j, x) : 0;
        unsigned long long take = __ballot(a32 >= floor32 && ahead(x, last));
        if (!take) break;
#pragma unroll 1
        for (; take; take &= take - 1) insert_cand(best, last, lane_cand(x, (int)__builtin_ctzll(take)), k);
      }
    }
    if (lane < k) sorted[wid][lane] = best;
    __syncthreads();
    if (lane < k && best.hi != 0) {
      int place = lane;
#pragma unroll 1
      for (int w = 0; w < nw; ++w) {
        if (w == wid) continue;
        int at = 0;
        while (at < k && ahead(sorted[w][at], best)) ++at;
        place += at;
      }
      if (place < k) put(best, place);
    }
    all = k;  // (there are more)
  }
  for (int i = all + tid; i < k; i += blockDim.x) {
    const int64_t at = (int64_t)g * k + i;
    c.scores_out[at] = -INFINITY;
    c.parents[at] = -1;
    c.tokens[at] = -1;
  }
}

struct BeamLayout {
  int nsplit, most, blocks;  // nsplit 0: by the live rows
  size_t live, part, keys;
};
BeamLayout beam_layout(int R, int W, int V, int k) {
  const int M = R * W;
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  BeamLayout L;
  L.most = std::max(1, std::min(kMaxLists / W, (V + kNW * kChunk - 1) / (kNW * kChunk)));
  L.nsplit = split_live(M, L.most);
  L.blocks = M * L.nsplit;
  // (where all rows' parts are the smallest already, dead rows leave nothing to the others)
  if (L.nsplit < L.most && M <= kLiveMax) {
    L.nsplit = 0;
    L.blocks = std::max(M, kBlocks);
  }
  if (L.nsplit > 0) L.most = L.nsplit;
  L.live = L.nsplit == 0 ? 256 : 0;
  L.part = up((size_t)M * L.most * sizeof(Part));
  L.keys = (size_t)M * L.most * k * sizeof(key_t);
  return L;
}

}  // namespace

size_t beam_ws_bytes(int R, int W, int V, int k) {
  const BeamLayout L = beam_layout(R, W, V, k);
  return L.live + L.part + L.keys;
}

int beam_launch(const BeamCall& c, hipStream_t st) {
  const BeamLayout L = beam_layout(c.R, c.W, c.V, c.k);
  BeamArgs a;
  a.c = c;
  a.nsplit = L.nsplit;
  a.most = L.most;
  char* ws = static_cast<char*>(c.ws);
  a.live = reinterpret_cast<int32_t*>(ws);
  a.part = reinterpret_cast<Part*>(ws + L.live);
  a.keys = reinterpret_cast<key_t*>(ws + L.live + L.part);
  const dim3 grid((uint32_t)L.blocks);
  if (c.dtype == Q35_F32) hipLaunchKernelGGL(beam_score_kernel<Q35_F32>, grid, dim3(kT), 0, st, a);
  else if (c.dtype == Q35_F16) hipLaunchKernelGGL(beam_score_kernel<Q35_F16>, grid, dim3(kT), 0, st, a);
  else hipLaunchKernelGGL(beam_score_kernel<Q35_BF16>, grid, dim3(kT), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  // a thread per list, and a wave per beam for the sums
  const int waves = std::max(1, std::min(kJoinWaves, std::max(c.W, (c.W * L.most + 63) / 64)));
  hipLaunchKernelGGL(beam_join_kernel, dim3(c.R), dim3(waves * 64), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

}  // namespace q35

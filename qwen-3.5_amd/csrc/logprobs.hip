// Scores of rows of logits: log probability and rank of a given token, entropy, highest alternatives.
//
// One pass over each row.  With d = x - m (m the running maximum) a lane keeps S = sum e^d and
// U = sum d e^d of what it has seen; when m rises by c, U becomes (U - c S) e^-c and S becomes S e^-c,
// so that at the end lse = m + ln S and the entropy is -sum p ln p = ln S - U / S, both from numbers
// of the size of the result (never as a difference of two lse-sized ones).  The rank of the
// target counts the values ranked before it in the same pass; its logit is one load at the start.
//
// The alternatives: each wave's list (toplist.h).  Waves, then the splits of a row (blocks), are joined by ranks: a
// key's place is the number of larger keys.
#include "toplist.h"

#include <algorithm>
#include <cmath>

namespace q35 {

namespace {

constexpr int kT = 256;         // threads per block
constexpr int kNW = kT / 64;
constexpr int kMaxSplit = 256;  // blocks per row: the joining block holds one part's sums per thread
constexpr int kLevels = 7;      // of the join's floors: 2^6 = kMaxTop
constexpr int kMaxCand = kLevels * kMaxTop;  // sum over i of 2^i ceil(top / 2^i), 2^i <= top

struct ScoreArgs {
  ScoreCall c;
  int32_t nsplit, len;  // values per split
  float* stat;          // [M][nsplit][4]: m, S, U, -
  int32_t* cnt;         // [M][nsplit]: values ranked before the target
  key_t* keys;          // [M][nsplit][top]
};

// running maximum, sum and weighted sum of a lane
struct Stat {
  float m, s, u;
};
Q35_DEV void stat_join(Stat& a, float m, float s, float u) {
  const float mn = fmaxf(a.m, m);
  const float r = mn == -INFINITY ? 0.f : mn;
  const float da = fmaxf(a.m - r, -1e4f), db = fmaxf(m - r, -1e4f);
  const float ea = exp_d(da), eb = exp_d(db);
  a.u = (a.u + da * a.s) * ea + (u + db * s) * eb;
  a.s = a.s * ea + s * eb;
  a.m = mn;
}

// ln S, S >= 1 (the maximum's own term is 1): the exponent apart from the rest f in [1, 2), whose logarithm is off by a
// few 2^-24 of itself, and what f loses in f32.  So ln 1 is 0, and no log probability comes out above 0.
// (With the f64 functions, whose code every block fetches, and the lists asked for only when wanted, the join
// took 7.2 us; 5.1 so.)
Q35_DEV double ln_sum(double S) {
  int e;
  const double f = 2.0 * frexp(S, &e);
  const float g = (float)f;
  return ((double)(e - 1) + (double)__builtin_amdgcn_logf(g)) * 0.693147180559945309 + (double)((float)(f - (double)g) * __builtin_amdgcn_rcpf(g));
}
// Final numbers of row m of the call; l = ln S.
Q35_DEV void finish_row(const ScoreCall& c, int m, float mx, double S, double U, double l, int cnt) {
  if (c.entropy) c.entropy[m] = S > 0.0 ? fmaxf((float)l - (float)U / (float)S, 0.f) : S == 0.0 ? 0.f : NAN;
  if (!c.targets) return;
  const int t = c.targets[m];
  if (t < 0 || t >= c.V) {
    c.logprob[m] = t < 0 ? 0.f : NAN;
    c.rank[m] = -1;
    if (t >= c.V) raise_status(c.status, Q35_STATUS_ARG);
    return;
  }
  const int64_t o = (int64_t)m * c.ld + t;
  const float x = c.dtype == Q35_F32 ? value<Q35_F32>(c.x, o) : c.dtype == Q35_F16 ? value<Q35_F16>(c.x, o) : value<Q35_BF16>(c.x, o);
  c.logprob[m] = mx == -INFINITY && S == 0.0 ? -INFINITY : (float)((double)(x - mx) - l);
  c.rank[m] = cnt;
}
Q35_DEV void put_top(const ScoreCall& c, int m, int i, key_t k, float mx, double S, double l) {
  const int64_t o = (int64_t)m * c.top + i;
  c.top_ids[o] = key_index(k);
  const float x = from_asc((uint32_t)(k >> 32));
  c.top_lp[o] = mx == -INFINITY && S == 0.0 ? -INFINITY : (float)((double)(x - mx) - l);
}

// Blocks (row, split).  Bound by the stream for many rows (700 rows of 248320 f32 values, top 5: 120 us, 5.8 TB/s; 1500
// rows 6.2; loads alone 6.7), beside 13 vector instructions per 64 values, half of them the exponential and its
// sums; by round trips and code that every block fetches for one row (10 us).
template <int DT>
__global__ __launch_bounds__(kT) void score_kernel(const ScoreArgs a) {
  const ScoreCall& c = a.c;
  __shared__ key_t lists[kNW][kMaxTop];
  __shared__ key_t buf[kNW][64];
  __shared__ float stage[kNW][kPer][64];
  __shared__ float sm[kNW], ss[kNW], su[kNW];
  __shared__ int sc[kNW];
  __shared__ key_t block_last;  // the largest of the waves' last wanted keys
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int m = blockIdx.x / a.nsplit, sp = blockIdx.x % a.nsplit;
  constexpr int kEs = DT == Q35_F32 ? 4 : 2, kVec = 16 / kEs;  // values of a 16-byte load
  const char* row = static_cast<const char*>(c.x) + (int64_t)m * c.ld * kEs;
  // index i of the row is value i + shift of the 16-byte words that begin at or before it
  const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / kEs);
  const char* base = row - shift * kEs;
  const int i0 = sp * a.len, i1 = min(c.V, i0 + a.len);  // the split's values
  int tgt = -1;
  float xt = 0.f;
  if (c.targets) {
    tgt = c.targets[m];
    if (tgt >= 0 && tgt < c.V) xt = value<DT>(row, tgt);
    else tgt = -1;
  }
  // the next float above it (NaN above +inf: nothing is >= that)
  const uint32_t xb = __float_as_uint(xt + 0.0f);
  const float above = __uint_as_float(xt == 0.f ? 1u : (xb & 0x80000000u) ? xb - 1u : xb + 1u);
  Stat st = {-INFINITY, 0.f, 0.f};
  int cnt = 0;  // (the wave's)
  key_t best = 0, last = 0;  // the lane's key of the wave's list; what a value must pass to get in
  const int top = c.top;
  const int w_first = (i0 + shift) / kVec, w_end = (i1 + shift + kVec - 1) / kVec;  // words of the split
  constexpr int kWords = kPer / kVec;
  constexpr uint32_t kAll = (1u << kPer) - 1u;
  bool first = true;
  if (top > 0) {
    if (tid == 0) block_last = 0;
    __syncthreads();
  }
  for (int w0 = w_first + wid * (kChunk / kVec); w0 < w_end; w0 += kNW * (kChunk / kVec)) {
    float x[kPer];
    uint32_t ok = kAll;  // which of the values belong to the split
    const int f0 = w0 * kVec - shift;  // the chunk's first index
    const bool whole = f0 >= i0 && f0 + kChunk <= i1;  // (uniform in the wave)
    auto index = [&](int e) { return f0 + (e / kVec * 64 + lane) * kVec + e % kVec; };
    if (whole) {
      uint4 v[kWords];
#pragma unroll
      for (int g = 0; g < kWords; ++g) v[g] = ldg16_nt(base + (int64_t)w0 * 16 + (g * 64 + lane) * 16);
#pragma unroll
      for (int g = 0; g < kWords; ++g) {
        const uint32_t d[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          x[g * kVec + j] = DT == Q35_F32 ? __uint_as_float(d[j & 3]) : half_of<DT>(d[(j >> 1) & 3], j & 1);
      }
    } else {  // (its words may hold others' values too)
      ok = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int f = index(e);
        const float v = value<DT>(row, min(max(f, i0), i1 - 1));
        const bool in = f >= i0 && f < i1;
        x[e] = in ? v : -INFINITY;
        ok |= (in ? 1u : 0u) << e;
      }
    }
    // (a wave by itself would find one of its `top` highest values in half of the chunks of a long row)
    const key_t bl = top > 0 ? __hip_atomic_load(&block_last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : 0;
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) mx = fmaxf(mx, x[e]);
    {
      const float mn = fmaxf(st.m, mx);
      const float r = mn == -INFINITY ? 0.f : mn;
      const float dc = fmaxf(st.m - r, -1e4f), ec = exp_d(dc);
      st.u = (st.u + dc * st.s) * ec;
      st.s *= ec;
      st.m = mn;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float d = x[e] - r, p = exp_d(d);
        st.s += p;
        st.u += fmaxf(d, -1e4f) * p;
      }
    }
    if (tgt >= 0) {
      // a chunk before the target's counts what is >= it, one behind it what is >= the next float; the chunk in
      // which it lies, chunks with others' values and a NaN go by the keys
      if (xt != xt || !whole || (uint32_t)(tgt - f0) < (uint32_t)kChunk) {
        const key_t kt = key_of(xt, tgt);
#pragma unroll
        for (int e = 0; e < kPer; ++e) cnt += __popcll(__ballot(key_of(x[e], index(e)) > kt && ((ok >> e) & 1u)));
      } else {
        const float from = f0 < tgt ? xt : above;
#pragma unroll
        for (int e = 0; e < kPer; ++e) cnt += __popcll(__ballot(x[e] >= from));
      }
    }
    if (top > 0) list_chunk(x, mx, ok, whole, index, bl, first, best, last, top, stage[wid], buf[wid], &block_last);
  }
  // lanes, then waves
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(st.m, o, 64), os = __shfl_xor(st.s, o, 64), ou = __shfl_xor(st.u, o, 64);
    stat_join(st, om, os, ou);
  }
  if (lane == 0) {
    sm[wid] = st.m;
    ss[wid] = st.s;
    su[wid] = st.u;
    sc[wid] = cnt;
  }
  if (top > 0) lists[wid][lane] = best;
  __syncthreads();
  Stat all = {sm[0], ss[0], su[0]};
  int before = sc[0];
#pragma unroll
  for (int w = 1; w < kNW; ++w) {
    stat_join(all, sm[w], ss[w], su[w]);
    before += sc[w];
  }
  const int64_t slot = (int64_t)m * a.nsplit + sp;
  if (tid == 0) {
    if (a.nsplit == 1) {
      finish_row(c, m, all.m, (double)all.s, (double)all.u, ln_sum((double)all.s), before);
    } else {
      float* o = a.stat + slot * 4;
      o[0] = all.m;
      o[1] = all.s;
      o[2] = all.u;
      a.cnt[slot] = before;
    }
  }
  if (top > 0 && lane < top) {
    // the key's place among the block's: its own list's keys before it, and the other lists' larger ones
    int at[kNW] = {};
#pragma unroll 1
    for (int step = 1 << (31 - __clz(top)); step > 0; step >>= 1) {  // (the lists' searches side by side)
#pragma unroll
      for (int w = 0; w < kNW; ++w)
        if (at[w] + step <= top && lists[w][at[w] + step - 1] > best) at[w] += step;
    }
    int place = 0;  // (its own list's larger keys are those of the lanes before it)
#pragma unroll
    for (int w = 0; w < kNW; ++w) place += at[w];
    if (best != 0 && place < top) {
      if (a.nsplit == 1) put_top(c, m, place, best, all.m, (double)all.s, ln_sum((double)all.s));
      else a.keys[slot * top + place] = best;
    }
    // a split with fewer values than `top` leaves the rest of its list empty
    const int have = min(top, i1 - i0);
    if (a.nsplit > 1 && wid == 0 && lane >= have) a.keys[slot * top + lane] = 0;
  }
}

// Block per row: joins its splits.  6 us (61 splits of 20 keys), round trips.
__global__ __launch_bounds__(kT) void score_join_kernel(const ScoreArgs a) {
  const ScoreCall& c = a.c;
  __shared__ key_t cand[kMaxCand];
  __shared__ key_t heads[kLevels * kMaxSplit];
  __shared__ key_t floors[kLevels];
  __shared__ float sm[kT];
  __shared__ double sS[kNW], sU[kNW];
  __shared__ int sn[kNW];
  __shared__ int ncand;
  const int m = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, ns = a.nsplit, top = c.top;
  const float* stat = a.stat + (int64_t)m * ns * 4;
  const bool in = tid < ns;
  // (the lists' first keys are asked for with everything else)
  const key_t* ks = a.keys + (int64_t)m * ns * top;
  constexpr int kFirst = 8;
  key_t kf[kFirst];
#pragma unroll
  for (int i = 0; i < kFirst; ++i) kf[i] = tid + i * kT < ns * top ? ks[tid + i * kT] : 0;
  const float mi = in ? stat[tid * 4] : -INFINITY, si = in ? stat[tid * 4 + 1] : 0.f, ui = in ? stat[tid * 4 + 2] : 0.f;
  int n = in ? a.cnt[(int64_t)m * ns + tid] : 0;
  float mx = mi;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) sm[wid] = mx;
  // level i: the 2^i-th key of every split
  const int levels = top > 0 ? 32 - __clz(top) : 0;
  const int lg = ns <= 64 ? 6 : 8, sp = tid & ((1 << lg) - 1);  // (a wave per level, or the block)
  for (int i = tid >> lg; i < levels; i += kT >> lg) heads[i << lg | sp] = sp < ns ? ks[sp * top + (1 << i) - 1] : 0;
  if (tid < kLevels) floors[tid] = 0;
  if (tid == 0) ncand = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kNW; ++w) mx = fmaxf(mx, sm[w]);
  const float r = mx == -INFINITY ? 0.f : mx;
  const float d = fmaxf(mi - r, -1e4f), e = exp_d(d);
  double S = (double)si * (double)e, U = ((double)ui + (double)d * (double)si) * (double)e;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    S += __shfl_xor(S, o, 64);
    U += __shfl_xor(U, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if (lane == 0) {
    sS[wid] = S;
    sU[wid] = U;
    sn[wid] = n;
  }
  // If r splits have 2^i keys at or above k, and 2^i r >= top, nothing below k counts; the largest such k of all
  // levels leaves few: of the 2^i-th keys at most ceil(top / 2^i) pass, each with at most 2^i keys of its list
  // down to the next level's, so kMaxCand in all, wherever in the row the largest values lie.
  for (int i = tid >> lg; i < levels; i += kT >> lg) {
    const key_t* row = heads + (i << lg);
    const key_t h = row[sp];
    int before = 0;
#pragma unroll 8
    for (int s = 0; s < 64; ++s) before += row[s] > h ? 1 : 0;
    if (lg > 6) {
      for (int s = 64; s < ns; ++s) before += row[s] > h ? 1 : 0;
    }
    if (h != 0 && before == (top - 1) >> i) floors[i] = h;
  }
  __syncthreads();
  S = (sS[0] + sS[1]) + (sS[2] + sS[3]);
  U = (sU[0] + sU[1]) + (sU[2] + sU[3]);
  n = (sn[0] + sn[1]) + (sn[2] + sn[3]);
  const double l = ln_sum(S);
  if (tid == 0) finish_row(c, m, mx, S, U, l, n);
  if (top == 0) return;
  key_t fl = 0;
#pragma unroll
  for (int i = 0; i < kLevels; ++i) fl = floors[i] > fl ? floors[i] : fl;
#pragma unroll
  for (int i = 0; i < kFirst; ++i)
    if (kf[i] != 0 && kf[i] >= fl) cand[atomicAdd(&ncand, 1)] = kf[i];
  for (int q = tid + kFirst * kT; q < ns * top; q += kT) {
    const key_t k = ks[q];
    if (k != 0 && k >= fl) cand[atomicAdd(&ncand, 1)] = k;
  }
  __syncthreads();
  const int nc = ncand;
  for (int q = tid; q < nc; q += kT) {
    const key_t k = cand[q];
    int place = 0;
    for (int s = 0; s < nc; ++s) place += cand[s] > k ? 1 : 0;
    if (place < top) put_top(c, m, place, k, mx, S, l);
  }
}

constexpr int kBlocks = 4 * 256;
// Blocks per row: enough to fill the chip when rows are few, of one chunk per wave at least (248320 values, up to
// 1024, 512 or 256 blocks: 64 rows 22, 25, 31 us; 400 rows 72, 77, 96; 2048 blocks: 700 rows 136 us instead of 122).
int score_split(int M, int V) {
  const int want = (kBlocks + M - 1) / M, most = std::min(kMaxSplit, (V + kNW * kChunk - 1) / (kNW * kChunk));
  return std::max(1, std::min(want, most));
}

struct ScoreLayout {
  int nsplit;
  size_t stat, cnt, keys;
};
ScoreLayout score_layout(int M, int V, int top) {
  ScoreLayout L;
  L.nsplit = score_split(M, V);
  const size_t n = L.nsplit > 1 ? (size_t)M * L.nsplit : 0;
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  L.stat = up(n * 16);
  L.cnt = up(n * 4);
  L.keys = up(n * top * 8);
  return L;
}

}  // namespace

size_t token_logprobs_ws_bytes(int M, int V, int top) {
  const ScoreLayout L = score_layout(M, V, top);
  return L.stat + L.cnt + L.keys;
}

int token_logprobs_launch(const ScoreCall& c, hipStream_t st) {
  const ScoreLayout L = score_layout(c.M, c.V, c.top);
  ScoreArgs a;
  a.c = c;
  a.nsplit = L.nsplit;
  a.len = (c.V + L.nsplit - 1) / L.nsplit;
  char* ws = static_cast<char*>(c.ws);
  a.stat = reinterpret_cast<float*>(ws);
  a.cnt = reinterpret_cast<int32_t*>(ws + L.stat);
  a.keys = reinterpret_cast<key_t*>(ws + L.stat + L.cnt);
  const dim3 grid((uint32_t)c.M * L.nsplit);
  if (c.dtype == Q35_F32) hipLaunchKernelGGL(score_kernel<Q35_F32>, grid, dim3(kT), 0, st, a);
  else if (c.dtype == Q35_F16) hipLaunchKernelGGL(score_kernel<Q35_F16>, grid, dim3(kT), 0, st, a);
  else hipLaunchKernelGGL(score_kernel<Q35_BF16>, grid, dim3(kT), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  if (L.nsplit > 1) {
    hipLaunchKernelGGL(score_join_kernel, dim3(c.M), dim3(kT), 0, st, a);
    Q35_HIP_TRY(hipGetLastError());
  }
  return Q35_OK;
}

}  // namespace q35

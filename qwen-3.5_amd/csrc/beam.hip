// The next beams of groups of beams: of all continuations (beam w, token v) of a group the k with the highest
// score[w] + x[w][v] - ln sum e^x[w].
//
// In a row the sum of the logarithm is the same for all tokens, so a row's best continuations are its highest
// logits.  One pass over the logits (blocks (row, part)) keeps each part's k highest and its maximum m and sum
// S of e^(x - m); a block per group then forms the rows' logarithms and chooses among the parts' lists.  Rows that
// have ended or whose beam is dead are not read.
// Continuations of different beams lie close together, and which ones are chosen must not hang on a rounding: sums over
// lanes and parts, logarithms and scores are f64, and the f32 exponentials' own errors (2^-23 each) mean out over the
// terms that matter: two beams' scores change places if they lie within about 10^-8.
#include "toplist.h"

#include <algorithm>

namespace q35 {

namespace {

constexpr int kT = 256;
constexpr int kNW = kT / 64;
constexpr int kMaxSplit = 256;
constexpr int kJoinWaves = 16;

struct alignas(16) Part {
  double s;
  float m, pad;
};
struct BeamArgs {
  BeamCall c;
  int32_t nsplit, len;  // values per part
  Part* part;           // [R W][nsplit]
  key_t* keys;          // [R W][nsplit][k]
};

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
  const int row_i = blockIdx.x / a.nsplit, sp = blockIdx.x % a.nsplit;
  if (beam_state(c, row_i) != kLive) return;
  constexpr int kEs = DT == Q35_F32 ? 4 : 2, kVec = 16 / kEs;
  const char* row = static_cast<const char*>(c.x) + (int64_t)row_i * c.ld * kEs;
  const int i0 = sp * a.len, i1 = min(c.V, i0 + a.len);
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
  const int64_t slot = (int64_t)row_i * a.nsplit + sp;
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

// A continuation: its score's bits in ascending order, and its number w V + v in the group; hi 0: none
struct Cand {
  unsigned long long hi;
  uint32_t ix;
};
Q35_DEV bool ahead(const Cand& a, const Cand& b) { return a.hi > b.hi || (a.hi == b.hi && a.ix < b.ix); }
Q35_DEV unsigned long long asc64(double c) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, c + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
Q35_DEV double from_asc64(unsigned long long a) { return __builtin_bit_cast(double, a >> 63 ? a & ~(1ull << 63) : ~a); }
Q35_DEV Cand lane_cand(const Cand& c, int lane) {
  return Cand{lane_key(c.hi, lane), (uint32_t)__builtin_amdgcn_readlane((int)c.ix, lane)};
}
// Puts c (the same in every lane) into the sorted list that the lanes hold; last: its top-th
Q35_DEV void insert_cand(Cand& best, Cand& last, const Cand& c, int top) {
  if (!ahead(c, last)) return;
  const Cand up = {((unsigned long long)(uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(best.hi >> 32), 0x138, 0xf, 0xf, false) << 32) |
                       (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(uint32_t)best.hi, 0x138, 0xf, 0xf, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best.ix, 0x138, 0xf, 0xf, false)};
  // a place takes the first of what it has and of the second of c and the one before it
  const Cand in = ahead(up, c) ? c : up;
  if (ahead(in, best)) best = in;
  if ((int)(threadIdx.x & 63) >= top) best = Cand{0, ~0u};
  last = lane_cand(best, top - 1);
}

// Block per group.
__global__ __launch_bounds__(kJoinWaves * 64) void beam_join_kernel(const BeamArgs a) {
  const BeamCall& c = a.c;
  __shared__ double off[kMaxBeams];
  __shared__ int state[kMaxBeams];
  __shared__ unsigned long long lhi[kJoinWaves][kMaxTop];
  __shared__ uint32_t lix[kJoinWaves][kMaxTop];
  __shared__ uint32_t bound;  // the highest f32 score, as bits in ascending order, that k continuations are known to reach
  __shared__ int found[kJoinWaves];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x / 64;
  const int g = blockIdx.x, W = c.W, ns = a.nsplit, k = c.k, nl = W * ns;
  const int64_t row0 = (int64_t)g * W;
  constexpr int kAhead = 4;
  const key_t* keys = a.keys + row0 * ns * k;
  key_t pre[kAhead];
  auto load = [&](int l, int j0) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) pre[e] = l < nl && j0 + e < k ? keys[(int64_t)l * k + j0 + e] : 0;
  };
  load(wid * 64 + lane, 0);
  if (tid == 0) bound = 0;
  for (int w = wid; w < W; w += nw) {
    const int row = (int)row0 + w, st = beam_state(c, row);
    double o = c.scores[row];
    if (st == kLive) {
      float m = -INFINITY;
      for (int i = lane; i < ns; i += 64) m = fmaxf(m, a.part[(int64_t)row * ns + i].m);
#pragma unroll
      for (int e = 32; e > 0; e >>= 1) m = fmaxf(m, __shfl_xor(m, e, 64));
      const float r = m == -INFINITY ? 0.f : m;
      double S = 0.0;
      for (int i = lane; i < ns; i += 64) {
        const Part p = a.part[(int64_t)row * ns + i];
        S += p.s * exp_near(p.m - r);
      }
#pragma unroll
      for (int e = 32; e > 0; e >>= 1) S += __shfl_xor(S, e, 64);
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
  Cand best = {0, ~0u}, last = {0, ~0u};
  bool seeded = false;
  for (int l0 = wid * 64; l0 < nl; l0 += nw * 64) {
    const int l = l0 + lane, w = l < nl ? l / ns : 0, sp = l - w * ns;
    const int st = l < nl ? state[w] : kDead;
    const double o = off[w];
    if (l0 != wid * 64) load(l, 0);
    for (int j0 = 0; j0 < k; j0 += kAhead) {
      if (j0 > 0) load(l, j0);
      bool more = true;
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const key_t key = pre[e];
        double s = -INFINITY;
        uint32_t ix = 0;
        if (st == kLive && key != 0) {
          s = o + (double)from_asc((uint32_t)(key >> 32));
          ix = (uint32_t)w * (uint32_t)c.V + (uint32_t)key_index(key);
        } else if (st == kEnded && sp == 0 && j0 + e == 0) {
          s = o;
          ix = (uint32_t)w * (uint32_t)c.V + (uint32_t)c.ended[row0 + w];
        }
        const bool some = s > -INFINITY;
        const Cand x = {some ? asc64(s) : 0, ix};
        const uint32_t a32 = some ? asc((float)s) : 0;
        if (!seeded) {
          // (float is monotonic: what is below the k-th largest of the lanes' floats is not among the k)
          seeded = true;
          const uint32_t t = (uint32_t)(seed_key(some ? (float)s : -INFINITY, k) >> 32) + 1u;
          if (t > 1 && lane == 0) atomicMax(&bound, t);
        }
        const uint32_t b = __hip_atomic_load(&bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        unsigned long long take = __ballot(some && a32 >= b && ahead(x, last));
        if (!take) {  // (lists fall: nothing behind these is wanted either)
          more = false;
          break;
        }
        for (; take; take &= take - 1) insert_cand(best, last, lane_cand(x, (int)__builtin_ctzll(take)), k);
        if (last.hi != 0 && lane == 0) atomicMax(&bound, asc((float)from_asc64(last.hi)));
      }
      if (!more) break;
    }
  }
  if (lane < k) {
    lhi[wid][lane] = best.hi;
    lix[wid][lane] = best.ix;
  }
  const int have = __popcll(__ballot(best.hi != 0));
  if (lane == 0) found[wid] = have;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < nw; ++w) all += found[w];
  if (lane < have) {
    int place = lane;
    for (int w = 0; w < nw; ++w) {
      if (w == wid) continue;
      int at = 0;
      for (int step = 1 << (31 - __clz(k)); step > 0; step >>= 1)
        if (at + step <= found[w] && ahead(Cand{lhi[w][at + step - 1], lix[w][at + step - 1]}, best)) at += step;
      place += at;
    }
    if (place < k) {
      const int64_t at = (int64_t)g * k + place;
      const uint32_t w = best.ix / (uint32_t)c.V;
      c.scores_out[at] = (float)from_asc64(best.hi);
      c.parents[at] = (int32_t)(row0 + w);
      c.tokens[at] = (int32_t)(best.ix - w * (uint32_t)c.V);
    }
  }
  for (int i = all + tid; i < k; i += blockDim.x) {
    const int64_t at = (int64_t)g * k + i;
    c.scores_out[at] = -INFINITY;
    c.parents[at] = -1;
    c.tokens[at] = -1;
  }
}

// Parts per row: as token_logprobs's splits, enough to fill the chip when rows are few
constexpr int kBlocks = 4 * 256;
int beam_split(int M, int V) {
  const int want = (kBlocks + M - 1) / M, most = std::min(kMaxSplit, (V + kNW * kChunk - 1) / (kNW * kChunk));
  return std::max(1, std::min(want, most));
}
size_t part_bytes(int M, int ns) { return ((size_t)M * ns * sizeof(Part) + 255) & ~(size_t)255; }

}  // namespace

size_t beam_ws_bytes(int R, int W, int V, int k) {
  const int ns = beam_split(R * W, V);
  return part_bytes(R * W, ns) + (size_t)R * W * ns * k * sizeof(key_t);
}

int beam_launch(const BeamCall& c, hipStream_t st) {
  const int M = c.R * c.W;
  BeamArgs a;
  a.c = c;
  a.nsplit = beam_split(M, c.V);
  a.len = (c.V + a.nsplit - 1) / a.nsplit;
  a.part = static_cast<Part*>(c.ws);
  a.keys = reinterpret_cast<key_t*>(static_cast<char*>(c.ws) + part_bytes(M, a.nsplit));
  const dim3 grid((uint32_t)M * a.nsplit);
  if (c.dtype == Q35_F32) hipLaunchKernelGGL(beam_score_kernel<Q35_F32>, grid, dim3(kT), 0, st, a);
  else if (c.dtype == Q35_F16) hipLaunchKernelGGL(beam_score_kernel<Q35_F16>, grid, dim3(kT), 0, st, a);
  else hipLaunchKernelGGL(beam_score_kernel<Q35_BF16>, grid, dim3(kT), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  // a wave per 64 lists, and one per beam for the sums
  const int waves = std::max(1, std::min(kJoinWaves, std::max(c.W, (c.W * a.nsplit + 63) / 64)));
  hipLaunchKernelGGL(beam_join_kernel, dim3(c.R), dim3(waves * 64), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

}  // namespace q35

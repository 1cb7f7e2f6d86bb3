// Rows of state tensors gathered by parent, in place or into other tensors: what a fork does with states that are
// one per sequence (DeltaNet's conv and recurrent states, contiguous caches, histories).
//
// In place, row j becomes what row parent[j] was, and a row may be overwritten and a parent of others, in chains and
// cycles.  Columns of the rows do not touch each other: a block takes a slab of columns of all rows that change, reads it
// into registers (up to 64 KB), waits for all of its reads, and writes.  So rows that stay are not read, nothing is copied
// twice, and no buffer is needed.
#include "pages.h"

#include <algorithm>

namespace q35 {

namespace {

constexpr int kT = 256;
constexpr int kPer = 16;  // words of a thread
constexpr int kStates = 64;

struct StatesArgs {
  q35_state s[kStates];
  const int32_t* parent;
  uint32_t* status;
  int32_t n, B, Bo, slab_log;  // log2 of the words of a slab at most
  int32_t copies;              // not in place: every row that has a parent is written
};

// words as they lie in memory and in registers
template <int kW>
struct Word;
template <>
struct Word<16> {
  typedef q35_u32x4 M, R;
};
template <>
struct Word<4> {
  typedef uint32_t M, R;
};
template <>
struct Word<1> {
  typedef uint8_t M;
  typedef uint32_t R;
};

// All blocks find the rows that change, then take the slabs of all states in turn.  Bound by HBM: 1.13 GB read and written
// in 220 us, 5.1 TB/s, a large copy's rate (through the caches 12 more; with half the words per thread, slabs of 512
// bytes a row, half as long again); 8 rows of 20 MB 13 us, 4 of 0.8 MB 6.7 us (launch, parents, a slab).  Into other tensors 5.7 TB/s.
template <int kW>
__global__ __launch_bounds__(kT) void states_fork_kernel(const StatesArgs a) {
  typedef typename Word<kW>::M M;
  typedef typename Word<kW>::R R;
  extern __shared__ int moves[];  // rows that change
  __shared__ int count[kT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int nm = 0;
  bool bad = false;
  for (int j0 = 0; j0 < a.Bo; j0 += kT) {
    const int j = j0 + tid;
    const int p = j < a.Bo ? a.parent[j] : -1;
    const bool out = p < -1 || p >= a.B, in = p >= 0 && !out && (a.copies || p != j);
    bad |= out;
    const unsigned long long mask = __ballot(in);
    if (lane == 0) count[wid] = __popcll(mask);
    __syncthreads();
    int at = nm + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) {
      at += w < wid ? count[w] : 0;
      nm += count[w];
    }
    if (in) moves[at] = j << 16 | p;  // (rows are below 2^12)
    __syncthreads();
  }
  if (bad && blockIdx.x == 0) raise_status(a.status, Q35_STATUS_ARG);
  if (nm == 0) return;
  // words of a slab: a power of two, so that all rows' slabs are at most kPer words of a thread
  const int lg = min(a.slab_log, 31 - __clz(kT * kPer / nm));
  const int words = nm << lg;
  int64_t first = 0;
  int s = 0;
  int64_t slabs = (a.s[0].row_bytes / kW + (1 << lg) - 1) >> lg;
  for (int64_t item = blockIdx.x;; item += gridDim.x) {
    while (item >= first + slabs) {
      first += slabs;
      if (++s == a.n) return;
      slabs = (a.s[s].row_bytes / kW + (1 << lg) - 1) >> lg;
    }
    const q35_state d = a.s[s];
    const int64_t w0 = (item - first) << lg, left = d.row_bytes / kW - w0;
    R v[kPer] = {};
    auto place = [&](int i, int64_t& src, int64_t& dst) {
      const int x = tid + i * kT, mv = moves[min(x >> lg, nm - 1)];
      const int64_t w = x & ((1 << lg) - 1);
      src = (int64_t)(mv & 0xffff) * d.src_stride + (w0 + min(w, left - 1)) * kW;
      dst = (int64_t)(mv >> 16) * d.dst_stride + (w0 + w) * kW;
      return x < words && w < left;
    };
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (i * kT < words) {
        int64_t src, dst;
        place(i, src, dst);
        v[i] = __builtin_nontemporal_load((const Q35_GLOBAL M*)((const char*)d.src + src));
      }
    }
    // every read of the slab has arrived before a write of it begins
#pragma unroll
    for (int i = 0; i < kPer; ++i) asm volatile("" : "+v"(v[i]));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (i * kT < words) {
        int64_t src, dst;
        if (place(i, src, dst)) __builtin_nontemporal_store((M)v[i], (Q35_GLOBAL M*)((char*)d.dst + dst));
      }
    }
  }
}

template <int kW>
int launch(StatesArgs& a, hipStream_t st) {
  int64_t row = 0;
  for (int i = 0; i < a.n; ++i) row += a.s[i].row_bytes / kW;
  // slabs enough for all blocks, of 256 bytes at least
  const int64_t blocks = 4 * (int64_t)device_cus();
  int lg = 0;
  while (lg < 12 && (((int64_t)kW << lg) < 256 || (row >> (lg + 1)) >= blocks)) ++lg;
  a.slab_log = lg;
  hipLaunchKernelGGL(states_fork_kernel<kW>, dim3((uint32_t)blocks), dim3(kT), (size_t)a.Bo * 4, st, a);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

}  // namespace

int states_fork_launch(const q35_state* states, int n, const int32_t* parent, int B, int Bo, bool copies, uint32_t* status, hipStream_t st) {
  // words of 16 bytes where all of a state's addresses allow them, else of 4, else bytes
  auto word = [](const q35_state& s) {
    const uint64_t all = reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) | (uint64_t)s.src_stride | (uint64_t)s.dst_stride | (uint64_t)s.row_bytes;
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
  };
  for (const int kw : {16, 4, 1}) {
    StatesArgs a;
    a.parent = parent;
    a.status = status;
    a.B = B;
    a.Bo = Bo;
    a.copies = copies;
    a.n = 0;
    for (int i = 0; i <= n; ++i) {
      if (a.n == kStates || (i == n && a.n > 0)) {
        const int rc = kw == 16 ? launch<16>(a, st) : kw == 4 ? launch<4>(a, st) : launch<1>(a, st);
        if (rc) return rc;
        a.n = 0;
      }
      if (i < n && states[i].row_bytes > 0 && word(states[i]) == kw) a.s[a.n++] = states[i];
    }
  }
  return Q35_OK;
}

}  // namespace q35

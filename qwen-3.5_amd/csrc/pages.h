// Paged caches, token scores, beams: calls between the C ABI (capi_paged.cpp) and the kernels.
#pragma once
#include <atomic>

#include "q35_internal.h"

namespace q35 {

constexpr int kPageHd = 256;            // head_dim
constexpr int kPageMaxPages = 1 << 18;  // pages of a pool that fork / compact / copy keep in LDS bitmaps
constexpr int kPageMaxSeqs = 4096;      // rows of a table in fork
constexpr int kPageMaxEntries = 1 << 26;  // of a page table in fork / compact (one block goes over them)
constexpr int kPageFewPairs = 256;      // pairs of a copy that its blocks check themselves
constexpr int kPageMaxHeads = 1024;     // query heads
constexpr int kPageMaxRep = 16;         // query heads per kv head
constexpr int kMaxLds = 150 * 1024;     // dynamic LDS that the kernels here ask for at most
constexpr int kMaxTop = 64;             // alternatives per row of token_logprobs, continuations per group of beam_select
constexpr int kMaxBeams = 256;          // of a group

constexpr int kQ4Row = kPageHd / 2 + kPageHd / 16;  // bytes of a Q35_Q4 row: codes, a word per 32 values

inline int elt_size(int dtype) { return dtype == Q35_F32 ? 4 : 2; }

// bytes that one token of one head has in a plane
__host__ __device__ inline int row_bytes(const q35_pages& P) {
  return P.dtype == Q35_Q4 ? kQ4Row : P.head_dim * (P.dtype == Q35_F32 ? 4 : 2);
}
// bytes of one page of one layer
__host__ __device__ inline size_t page_bytes(const q35_pages& P) { return (size_t)2 * P.kv_heads * P.page * row_bytes(P); }

// Lets a kernel's launches use more than 64 KB of dynamic LDS; asked once per kernel and device (the call
// takes as long as a third of a launch).
template <auto kKernel>
void allow_lds(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (bytes <= 48 * 1024 || hipGetDevice(&dev) != hipSuccess) return;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds) == hipSuccess)
    done.fetch_or(bit, std::memory_order_relaxed);
}

int check_pages(const q35_pages& P, const char* what);

// *status &= ~bits on the stream
int status_clear_launch(uint32_t* status, uint32_t bits, hipStream_t st);

int pages_copy_launch(const q35_pages& src, const q35_pages& dst, const int32_t* sid, const int32_t* did, int n,
                      uint32_t* status, uint8_t* ok, hipStream_t st);

struct ReadCall {
  q35_pages P;
  const int32_t *table, *row, *pos;
  int32_t layer, ld, B, n;
  void* out;
  uint32_t* status;
};
int pages_read_launch(const ReadCall& c, hipStream_t st);

struct ForkCall {
  q35_pages P;
  const int32_t *table, *len, *parent, *grow;
  int32_t ld, B, Bo;
  int32_t *table_out, *len_out, *refs;
  uint32_t* status;
};
int pages_fork_launch(const ForkCall& c, hipStream_t st);

struct CompactCall {
  q35_pages P;
  const int32_t* table;
  int32_t ld, B;
  int32_t *table_out, *refs, *used;
  uint32_t* status;
  int32_t* moves;  // ws: [n_pages] holes, [n_pages] movers
};
int pages_compact_launch(const CompactCall& c, hipStream_t st);

struct PagedAttn {
  q35_pages P;
  int32_t layer, nh, nkv, rot, T, B, ld_qg, ld_kv, ld_table, ld_out, rope_rows;
  float eps, scale;
  const float *qg, *k, *v, *qnw, *knw, *rcos, *rsin;
  const int32_t *start, *pos, *table;
  float* out;
  uint32_t* status;
  void* ws;
};
size_t paged_attn_ws_bytes(int nh, int nkv, int T, int B);
int paged_attn_launch(const PagedAttn& a, hipStream_t st);

struct ScoreCall {
  const void* x;
  int32_t dtype, M, V, top;
  int64_t ld;
  const int32_t* targets;
  float* logprob;
  int32_t* rank;
  float* entropy;
  int32_t* top_ids;
  float* top_lp;
  uint32_t* status;
  void* ws;
};
size_t token_logprobs_ws_bytes(int M, int V, int top);
int token_logprobs_launch(const ScoreCall& c, hipStream_t st);

struct BeamCall {
  const void* x;
  int32_t dtype, R, W, V, k;
  int64_t ld;
  const float* scores;
  const int32_t* ended;
  float* scores_out;
  int32_t *parents, *tokens;
  uint32_t* status;
  void* ws;
};
size_t beam_ws_bytes(int R, int W, int V, int k);
int beam_launch(const BeamCall& c, hipStream_t st);

// states: host; copies: dst is not src
int states_fork_launch(const q35_state* states, int n, const int32_t* parent, int B, int Bo, bool copies, uint32_t* status,
                       hipStream_t st);

Q35_DEV void raise_status(uint32_t* status, uint32_t bit) {
  if (status) __hip_atomic_fetch_or((Q35_GLOBAL uint32_t*)status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace q35

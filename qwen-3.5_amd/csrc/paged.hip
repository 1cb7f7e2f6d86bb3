// Attention of new tokens over a paged cache: q/k RMSNorm (1 + w), rotary, append of keys and values to
// the sequences' pages, causal softmax(q K^T / 16) V with shared kv heads, sigmoid output gate.
#include "pages.h"

#include <cmath>

namespace q35 {

namespace {

constexpr int kHd = kPageHd;
constexpr int kT = 256;

// The sequence of row t: b with start[b] <= t < start[b + 1]; false if there is none, or if its
// positions leave the table or the rotary rows (reported).
struct Seq {
  int b, i, n, p0;  // sequence, row within it, its rows, its cached tokens
};
Q35_DEV bool seq_ok(const PagedAttn& a, int n, int p0) {
  const int64_t cap = (int64_t)a.ld_table * a.P.page;
  const int64_t lim = cap < a.rope_rows ? cap : a.rope_rows;
  return p0 >= 0 && (int64_t)p0 + n <= lim;
}
Q35_DEV bool find_seq(const PagedAttn& a, int t, Seq* s, bool report) {
  int lo = 0, hi = a.B;  // the last b with start[b] <= t
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (a.start[m] <= t) lo = m;
    else hi = m;
  }
  const int s0 = a.start[lo], s1 = a.start[lo + 1];
  if (t < s0 || t >= s1) return false;
  s->b = lo;
  s->i = t - s0;
  s->n = s1 - s0;
  s->p0 = a.pos[lo];
  if (seq_ok(a, s->n, s->p0)) return true;
  if (report) raise_status(a.status, Q35_STATUS_ARG);
  return false;
}

// Byte offset of token p of row b's pages, plane 0, kv head 0; -1 if its page is not in the pool
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

Q35_DEV int64_t plane_elts(const PagedAttn& a) { return (int64_t)a.nkv * a.P.page * kHd; }
Q35_DEV int64_t page_elts(const PagedAttn& a) { return 2 * plane_elts(a); }

// wave sum in f64, the same in every lane
Q35_DEV double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// A key's value as the cache holds it: rounded to f32, then to the cache's type (both to nearest even).
// The empty asm keeps the compiler from rounding f64 to f16 in one step, as it otherwise does.
template <class E>
Q35_DEV E stored(double y) {
  float f = (float)y;
  asm("" : "+v"(f));
  return (E)f;
}

// Keys and values of the new tokens into their pages; a wave per (row, kv head).
template <int DT>
__global__ __launch_bounds__(kT) void paged_append_kernel(const PagedAttn a) {
  typedef typename Elt<DT>::T E;
  __shared__ double xs[kT / 64][kHd];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * (kT / 64) + wid;
  const int t = (int)(item / a.nkv), g = (int)(item % a.nkv);
  Seq s;
  const bool in = t < a.T && find_seq(a, t, &s, lane == 0);
  int page = -1, p = 0;
  if (in) {
    p = s.p0 + s.i;
    page = a.table[(int64_t)s.b * a.ld_table + p / a.P.page];
    if ((uint32_t)page >= (uint32_t)a.P.n_pages) {
      if (lane == 0) raise_status(a.status, Q35_STATUS_ARG);
      page = -1;
    }
  }
  const int d = 4 * lane;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (page >= 0) {
    const float4 k = *reinterpret_cast<const float4*>(a.k + (int64_t)t * a.ld_kv + (int64_t)g * kHd + d);
    v = *reinterpret_cast<const float4*>(a.v + (int64_t)t * a.ld_kv + (int64_t)g * kHd + d);
    const float4 w = *reinterpret_cast<const float4*>(a.knw + d);
    const double x0 = k.x, x1 = k.y, x2 = k.z, x3 = k.w;
    const double r = 1.0 / sqrt(wave_sum64((x0 * x0 + x1 * x1) + (x2 * x2 + x3 * x3)) / (double)kHd + (double)a.eps);
    xs[wid][d] = x0 * r * (1.0 + (double)w.x);
    xs[wid][d + 1] = x1 * r * (1.0 + (double)w.y);
    xs[wid][d + 2] = x2 * r * (1.0 + (double)w.z);
    xs[wid][d + 3] = x3 * r * (1.0 + (double)w.w);
  }
  __syncthreads();
  if (page < 0) return;
  const int half = a.rot / 2;
  E* kr = static_cast<E*>(a.P.data) + ((int64_t)a.layer * a.P.n_pages + page) * page_elts(a) +
          ((int64_t)g * a.P.page + p % a.P.page) * kHd;
  E* vr = kr + plane_elts(a);
  const float* cs = a.rcos + (int64_t)p * a.rot;
  const float* sn = a.rsin + (int64_t)p * a.rot;
  const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = d + j;
    double y = xs[wid][i];
    if (i < a.rot) {
      const double rh = i < half ? -xs[wid][i + half] : xs[wid][i - half];
      y = y * (double)cs[i] + rh * (double)sn[i];
    }
    kr[i] = stored<E>(y);
    vr[i] = (E)vv[j];
  }
}

// A wave per (row, query head), one key after another.
template <int DT>
__global__ __launch_bounds__(kT) void paged_attn_simple_kernel(const PagedAttn a) {
  typedef typename Elt<DT>::T E;
  __shared__ float xs[kT / 64][kHd];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * (kT / 64) + wid;
  const int t = (int)(item / a.nh), h = (int)(item % a.nh);
  Seq s;
  const bool in = t < a.T && find_seq(a, t, &s, false);
  const int d = 4 * lane;
  if (in) {
    const float4 q = *reinterpret_cast<const float4*>(a.qg + (int64_t)t * a.ld_qg + (int64_t)h * 2 * kHd + d);
    const float4 w = *reinterpret_cast<const float4*>(a.qnw + d);
    const float r = rsqrt_f(wave_sum(q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w) / (float)kHd + a.eps);
    xs[wid][d] = q.x * r * (1.0f + w.x);
    xs[wid][d + 1] = q.y * r * (1.0f + w.y);
    xs[wid][d + 2] = q.z * r * (1.0f + w.z);
    xs[wid][d + 3] = q.w * r * (1.0f + w.w);
  }
  __syncthreads();
  if (!in) return;
  const int p = s.p0 + s.i, half = a.rot / 2, g = h / (a.nh / a.nkv);
  float q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = d + j;
    q[j] = xs[wid][i];
    if (i < a.rot) {
      const float rh = i < half ? -xs[wid][i + half] : xs[wid][i - half];
      q[j] = q[j] * a.rcos[(int64_t)p * a.rot + i] + rh * a.rsin[(int64_t)p * a.rot + i];
    }
  }
  const E* base = static_cast<const E*>(a.P.data) + (int64_t)a.layer * a.P.n_pages * page_elts(a) + (int64_t)g * a.P.page * kHd;
  const int32_t* row = a.table + (int64_t)s.b * a.ld_table;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const float sl2 = a.scale * 1.44269504088896341f;
  for (int j = 0; j <= p; ++j) {
    int page = row[j / a.P.page];
    if ((uint32_t)page >= (uint32_t)a.P.n_pages) {
      if (lane == 0) raise_status(a.status, Q35_STATUS_ARG);
      page = 0;
    }
    const E* kr = base + (int64_t)page * page_elts(a) + (int64_t)(j % a.P.page) * kHd + d;
    const E* vr = kr + plane_elts(a);
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) x += q[e] * (float)kr[e];
    x = wave_sum(x) * sl2;
    const float mn = fmaxf(m, x);
    const float f = __builtin_amdgcn_exp2f(m - mn), pr = __builtin_amdgcn_exp2f(x - mn);
    m = mn;
    l = l * f + pr;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + pr * (float)vr[e];
  }
  const float4 gv = *reinterpret_cast<const float4*>(a.qg + (int64_t)t * a.ld_qg + (int64_t)h * 2 * kHd + kHd + d);
  float* dst = a.out + (int64_t)t * a.ld_out + (int64_t)h * kHd + d;
  *reinterpret_cast<float4*>(dst) = make_float4(o[0] / l * sigmoid_f(gv.x), o[1] / l * sigmoid_f(gv.y),
                                                o[2] / l * sigmoid_f(gv.z), o[3] / l * sigmoid_f(gv.w));
}

template <int DT>
int launch(const PagedAttn& a, hipStream_t st) {
  const int64_t ka = (int64_t)a.T * a.nkv, qa = (int64_t)a.T * a.nh;
  hipLaunchKernelGGL(paged_append_kernel<DT>, dim3((uint32_t)((ka + 3) / 4)), dim3(kT), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(paged_attn_simple_kernel<DT>, dim3((uint32_t)((qa + 3) / 4)), dim3(kT), 0, st, a);
  Q35_HIP_TRY(hipGetLastError());
  return Q35_OK;
}

}  // namespace

size_t paged_attn_ws_bytes(int nh, int nkv, int T, int B) {
  (void)nh; (void)nkv; (void)T; (void)B;
  return 256;
}

int paged_attn_launch(const PagedAttn& a, hipStream_t st) {
  return a.P.dtype == Q35_F32 ? launch<Q35_F32>(a, st) : a.P.dtype == Q35_F16 ? launch<Q35_F16>(a, st) : launch<Q35_BF16>(a, st);
}

}  // namespace q35

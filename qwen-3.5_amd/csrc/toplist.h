// The highest values of rows of logits, and their places: wave-wide sorted lists.
//
// A value and its index make one 64-bit key (the value's bits in ascending order,
// then the complement of the index), so "larger value, then lower index" is one unsigned comparison
// and every choice below is exact whatever the order of the work.  A wave keeps its best `top` keys
// sorted, one per lane; a chunk of values costs one comparison of each lane's maximum with the last wanted
// key, and only values above it are looked at: a few are put into the list one by one, many are put aside and
// joined with it, up to 64 at a time.  The waves of a block tell each other their last wanted keys.  The first
// chunk would have almost everything looked at: the last wanted key starts at the `top`-th of the 64 lanes'
// maxima instead (that many values are at least as large), or, for more than 32, the (top / 2)-th of their
// second largest values.
#pragma once
#include "pages.h"

namespace q35 {
namespace {

constexpr int kPer = 16;        // values of a lane per chunk
constexpr int kChunk = 64 * kPer;
constexpr int kFewKeys = 8;    // values of the lanes that are put into the list one by one

typedef unsigned long long key_t;

// a float's bits in ascending order; NaN below everything
Q35_DEV uint32_t asc(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
  return x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
Q35_DEV float from_asc(uint32_t a) {
  return a == 0 ? __uint_as_float(0x7fc00000u) : __uint_as_float((a & 0x80000000u) ? a & 0x7fffffffu : ~a);
}
Q35_DEV key_t key_of(float x, int i) { return ((key_t)asc(x) << 32) | (uint32_t)~i; }
Q35_DEV int key_index(key_t k) { return (int)~(uint32_t)k; }

Q35_DEV key_t lane_key(key_t k, int lane) {
  return ((key_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}

template <int DT>
Q35_DEV float value(const void* p, int64_t i) {
  if constexpr (DT == Q35_F32) return ((const Q35_GLOBAL float*)p)[i];
  if constexpr (DT == Q35_F16) return (float)((const Q35_GLOBAL _Float16*)p)[i];
  return __uint_as_float((uint32_t)((const Q35_GLOBAL uint16_t*)p)[i] << 16);
}
template <int DT>
Q35_DEV float half_of(uint32_t w, int h) {
  if constexpr (DT == Q35_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(h ? w >> 16 : w));
  return __uint_as_float(h ? w & 0xffff0000u : w << 16);
}

Q35_DEV float exp_d(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }

// What one lane of the wave wrote to LDS is read by others of the same wave.
Q35_DEV void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}
// The lanes' keys with `take` set behind the n of buf
Q35_DEV void push_keys(key_t* buf, int& n, key_t k, bool take) {
  const unsigned long long mask = __ballot(take);
  if (!mask) return;
  const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
  if (take) buf[at] = k;
  n += __popcll(mask);
}
// Joins the n <= 64 keys of buf with the sorted list that the lanes hold: a key's new place is the number of
// larger keys in both.  last becomes the list's top-th key.
Q35_DEV void merge_keys(key_t* buf, int n, key_t& best, key_t& last, int top) {
  const int lane = threadIdx.x & 63;
  wave_sync();
  const key_t c = lane < n ? buf[lane] : 0;
  int pc = 0, pb = lane;
  // (four at a time: the places behind the n and behind the list's `top` hold 0, which is larger than nothing)
  for (int j = 0; j < n; j += 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const key_t k = lane_key(c, j + e);
      pc += k > c ? 1 : 0;
      pb += k > best ? 1 : 0;
    }
  }
  if (lane_key(best, 0) != 0) {  // (the first time there is no list)
    for (int j = 0; j < top; j += 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) pc += lane_key(best, j + e) > c ? 1 : 0;
    }
  }
  wave_sync();
  buf[lane] = 0;
  wave_sync();
  // (empty places hold 0 and stay behind every key; only the first `top` places count)
  if (best != 0 && pb < top) buf[pb] = best;
  if (c != 0 && pc < top) buf[pc] = c;
  wave_sync();
  best = buf[lane];
  wave_sync();
  const key_t t = lane_key(best, top - 1);
  last = t > last ? t : last;
}

// Puts c into the sorted list that the lanes hold, if it is larger than its last wanted key.
Q35_DEV void insert_key(key_t& best, key_t& last, key_t c, int top) {
  if (c <= last) return;
  // a place takes the larger of its key and of the smaller of c and the key before it
  const key_t up = ((key_t)(uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(best >> 32), 0x138, 0xf, 0xf, false) << 32) |
                   (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)(uint32_t)best, 0x138, 0xf, 0xf, false);
  const key_t in = up < c ? up : c;
  best = (int)(threadIdx.x & 63) >= top ? 0 : in > best ? in : best;
  const key_t t = lane_key(best, top - 1);
  last = t > last ? t : last;
}

// What a key must pass, from one value of every lane (-inf or NaN: none): the r-th largest of them, without its
// lowest 6 bits (the lane's number takes their place, so that no two are equal); that many keys do.  0 if
// fewer lanes have one.
Q35_DEV key_t seed_key(float v, int r) {
  const uint32_t a = (v > -INFINITY ? asc(v) & ~63u : 0u) | (threadIdx.x & 63);
  int before = 0;
#pragma unroll 8
  for (int l = 0; l < 64; ++l) before += (uint32_t)__builtin_amdgcn_readlane((int)a, l) > a ? 1 : 0;
  const unsigned long long at = __ballot(before == r - 1);
  const uint32_t t = (uint32_t)__builtin_amdgcn_readlane((int)a, (int)__builtin_ctzll(at)) & ~63u;
  return t == 0 ? 0 : ((key_t)t << 32) - 1;
}

// A chunk of the wave's values: x[e] of index index(e), those whose bit of `ok` is set (all of them if `whole`), mx the lane's
// largest; bl: what the block's waves have found a value must pass.  stage, buf: the wave's LDS.
template <class Index>
Q35_DEV void list_chunk(const float (&x)[kPer], float mx, uint32_t ok, bool whole, Index index, key_t bl, bool& first, key_t& best,
                        key_t& last, int top, float (*stage)[64], key_t* buf, key_t* block_last) {
  const int lane = threadIdx.x & 63;
  if (first) {  // (uniform in the wave)
    first = false;
    last = seed_key(mx, top);
    if (top > 32) {  // second largest values: half of the lanes are enough
      float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float v = x[e] == x[e] ? x[e] : -INFINITY;  // (the smaller of a number and NaN is the number)
        m2 = fmaxf(m2, fminf(m1, v));
        m1 = fmaxf(m1, v);
      }
      const key_t l2 = seed_key(m2, (top + 1) / 2);
      last = l2 > last ? l2 : last;
    }
  }
  const key_t lb = lane_key(bl, 0);
  if (lb > last) last = lb;
  // values at or above the last wanted one (all, while that is nothing or NaN; a NaN always: its key decides)
  const uint32_t la = (uint32_t)(last >> 32);
  const float lf = la == 0 ? -INFINITY : from_asc(la);
  if (__ballot(!(mx < lf))) {
    uint32_t left = 0;  // the lane's values to look at
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e) left = left + left + (x[e] < lf ? 0u : 1u);
    left &= ok;
    // else a lane's only one is its largest (or NaN beside smaller numbers: too small either way)
    const bool stages = !whole || __ballot((left & (left - 1)) != 0) != 0;
    if (stages) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) stage[e][lane] = x[e];
      wave_sync();
    }
    const key_t before = last;
    // one of every lane at a time (a loop: written out for each of the 16 values, its code, which every
    // block fetches, took 0.6 us): a few are put into the list one by one, many are put aside and joined
    // with it, 64 at the most
    int n = 0;  // keys in buf
#pragma unroll 1
    for (;;) {
      const unsigned long long any = __ballot(left != 0);
      const int e = left != 0 ? __ffs(left) - 1 : 0;
      const key_t k = left != 0 ? key_of(stages ? stage[e][lane] : mx, index(e)) : 0;
      unsigned long long take = __ballot(k > last);
      if (n == 0 && __popcll(take) <= kFewKeys) {
        if (!any) break;
        for (; take; take &= take - 1) insert_key(best, last, lane_key(k, (int)__builtin_ctzll(take)), top);
        left &= left - 1;
      } else if (any ? n + __popcll(take) > 64 : n > 0) {
        merge_keys(buf, n, best, last, top);
        n = 0;  // (the same values again: fewer pass the list now)
      } else {
        push_keys(buf, n, k, k > last);
        left &= left - 1;
      }
    }
    wave_sync();
    if (last > before && lane == 0) __hip_atomic_fetch_max(block_last, last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
}

}  // namespace
}  // namespace q35

// b2q_paged.cuh -- what the paged attention's kernels share: 16-bit pairs, the
// requests' rows and the keys that a run of them sees.
#pragma once

#include "b2q_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2q {

constexpr int64_t kNowhere = -(int64_t{1} << 60);  // position of a padding row: before every key

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
}
// Either half of the pair is an infinity or a NaN.
template <bool BF16>
__device__ __forceinline__ bool nonfinite2(uint32_t u) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (u & e) == e || (u & (e << 16)) == (e << 16);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The new tokens of one request and the keys that a run of them can see.
struct Request {
  int64_t t0;     // first row of q
  int64_t n;      // new tokens
  int64_t len;    // keys the table can hold and the request has
  int64_t first;  // position of the first new token
};
__device__ __forceinline__ Request request_of(const PagedArgs& a, int b) {
  Request r;
  const int64_t lo = min(max(static_cast<int64_t>(a.cu_q[b]), int64_t{0}), a.T);
  const int64_t hi = min(max(static_cast<int64_t>(a.cu_q[b + 1]), lo), a.T);
  r.t0 = lo;
  r.n = min(hi - lo, a.max_q);
  const int64_t len = max(a.kv_len[b], 0);
  r.first = len - (hi - lo);
  r.len = min(len, a.width << a.page_shift);
  return r;
}
// Units of `unit` keys seen by some token at positions p_lo .. p_hi: the sinks'
// units 0 .. su - 1, then wu .. hu - 1.
struct Units {
  int64_t su, wu, hu;
  int64_t win_lo;  // first key of the window of p_lo
  __device__ __forceinline__ int64_t count() const { return su + (hu - wu); }
  __device__ __forceinline__ int64_t at(int64_t i) const { return i < su ? i : wu + (i - su); }
};
__device__ __forceinline__ Units units_of(const PagedArgs& a, int64_t len, int64_t p_lo, int64_t p_hi, int unit) {
  Units u;
  const int64_t hi = a.causal ? min(len, p_hi + 1) : len;
  u.hu = hi > 0 ? (hi + unit - 1) / unit : 0;
  u.win_lo = a.window > 0 ? max(int64_t{0}, p_lo - a.window + 1) : 0;
  u.wu = min(u.win_lo / unit, u.hu);
  const int64_t sk = a.window > 0 ? min(a.sinks, u.win_lo) : 0;
  u.su = min((sk + unit - 1) / unit, u.wu);
  return u;
}
__device__ __forceinline__ bool sees(const PagedArgs& a, int64_t p, int64_t j, int64_t len) {
  return j < len && (!a.causal || j <= p) && (a.window <= 0 || j > p - a.window || j < a.sinks);
}

// A key's infinite value makes the outputs of the rows that see it infinite, but in the tensor
// products it meets weights that are 0 where they have no bits left (an fp16 weight below 2^-25 of
// the largest, the rounding error of a weight that is exact) or negative (other rounding errors),
// and gives NaN.  So an output that is NaN although its row's sum is not is settled from the
// values themselves: a NaN, or infinities of both signs, among the keys that the row sees is NaN,
// else the infinity (none: the sums overflowed, NaN as before).  A row sees keys [lo, hi) and those
// of [0, sinks) below hi.  v: the kv head's values of page 0 at the first of 2 W columns; the
// result's bits x say that column x has an infinity or NaN of positive (.x) or negative (.y) sign,
// a NaN counting as both.  Rare, so the loop over the keys is plain.
template <int W, bool BF16>
__device__ __noinline__ uint2 nonfinite_seen(const uint16_t* v, const int32_t* table, int64_t n_pages, int page_shift,
                                             int64_t page_elems, int D, int lo, int hi, int sinks) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  uint2 seen = make_uint2(0u, 0u);
  for (int j = sinks > 0 ? 0 : lo; j < hi; j = j + 1 >= sinks && j + 1 < lo ? lo : j + 1) {
    const int32_t page = __ldg(table + (j >> page_shift));
    if (page < 0 || page >= n_pages) continue;
    const uint16_t* row = v + page * page_elems + static_cast<int64_t>(j & ((1 << page_shift) - 1)) * D;
    for (int w = 0; w < W; ++w) {
      const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(row) + w);
      if (!nonfinite2<BF16>(u)) continue;
      for (int x = 0; x < 2; ++x) {
        const uint32_t h = x ? u >> 16 : u & 0xffffu;
        if ((h & kExp) != kExp) continue;
        const bool nan = (h & 0x7fffu) != kExp;
        if (nan || h == kExp) seen.x |= 1u << (2 * w + x);
        if (nan || h != kExp) seen.y |= 1u << (2 * w + x);
      }
    }
  }
  return seen;
}
// What column x of a row with those bits is, where its sum gave NaN.
__device__ __forceinline__ float settled(uint2 seen, int x) {
  const bool up = (seen.x >> x) & 1u, down = (seen.y >> x) & 1u;
  return up == down ? NAN : up ? INFINITY : -INFINITY;
}

}  // namespace b2q

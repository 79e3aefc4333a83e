// b2q_lora.cu -- low-rank adapters of many requests beside a shared projection:
//   y[t] = resid[t] + scale_a * B_a (A_a x[t]),  a = the adapter of row t
// (rows of no adapter: y[t] = resid[t]).
//
// Plain form: a CTA has one tile of 16 sorted rows; a warp per value of A_a x,
// then a thread per column.
#include "b2q_groups.cuh"
#include "b2q_internal.h"

namespace b2q {

namespace {

constexpr int kTile = 16, kThreads = 256;

template <int X, int Y>
__global__ void __launch_bounds__(kThreads) lora_kernel(const LoraArgs a) {
  using XV = typename Val<X>::type;
  using YV = typename Val<Y>::type;
  __shared__ float h[kTile][kLoraMaxRank];
  __shared__ int row[kTile];
  const GroupTile t = find_group_tile(a.offsets, a.groups, a.T, blockIdx.x, kTile);
  if (t.group < 0) return;
  const int count = t.end - t.begin;
  if (threadIdx.x < kTile) {
    int r = -1;
    if (static_cast<int>(threadIdx.x) < count) {
      r = __ldg(a.order + t.begin + threadIdx.x);
      if (r < 0 || r >= a.T) r = -1;
    }
    row[threadIdx.x] = r;
  }
  __syncthreads();
  const bool live = t.group < a.groups;
  const int lane = threadIdx.x & 31;
  if (live) {
    const float scale = a.scales ? __ldg(a.scales + t.group) : 1.0f;
    for (int i = threadIdx.x >> 5; i < count * a.rank; i += kThreads / 32) {
      const int m = i / a.rank, r = i % a.rank;
      float sum = 0.0f;
      if (row[m] >= 0) {
        const XV* x = static_cast<const XV*>(a.x) + row[m] * a.ldx;
        const XV* w = static_cast<const XV*>(a.a) + (static_cast<int64_t>(t.group) * a.rank + r) * a.K;
        for (int64_t k = lane; k < a.K; k += 32) sum = fmaf(Val<X>::load(x + k), Val<X>::load(w + k), sum);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) h[m][r] = sum * scale;
    }
  }
  __syncthreads();
  for (int64_t n = threadIdx.x; n < a.N; n += kThreads)
    for (int m = 0; m < count; ++m) {
      if (row[m] < 0) continue;
      float sum = 0.0f;
      if (live) {
        const XV* w = static_cast<const XV*>(a.b) + (static_cast<int64_t>(t.group) * a.N + n) * a.rank;
        for (int r = 0; r < a.rank; ++r) sum = fmaf(Val<X>::load(w + r), h[m][r], sum);
      }
      sum += Val<Y>::load(static_cast<const YV*>(a.resid) + row[m] * a.ldr + n);
      static_cast<YV*>(a.y)[row[m] * a.ldy + n] = Val<Y>::to(sum);
    }
}

}  // namespace

cudaError_t launch_lora(const LoraArgs& a, int xtype, int ytype, int num_sms, cudaStream_t s) {
  (void)num_sms;
  void (*k)(const LoraArgs) = xtype == 1 ? (ytype == 0 ? lora_kernel<1, 0> : lora_kernel<1, 1>)
                                         : (ytype == 0 ? lora_kernel<2, 0> : lora_kernel<2, 2>);
  k<<<static_cast<unsigned>(a.T / kTile + a.groups + 1), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace b2q

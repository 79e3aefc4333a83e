// b2q_verify.cu -- which drafted tokens a target model keeps, and the token
// that follows them, from given random numbers (speculative sampling):
//   draft i of a request, token d, stays while  u_i q_i(d) < p_i(d)
//   the first that does not is replaced by a draw from w = max(p_i - q_i, 0)
//   (from p_i where that is 0 everywhere); after the last draft, from p's last row
//   the draw: the first token j with  w_0 + .. + w_j > v (w_0 + ... )
// Products, differences and sums are in 64 bits: in 32 the borders between the
// tokens of a large vocabulary would move by more than a rare token is wide.
//
// A cluster of CTAs has one request: each looks at the drafts itself (a warp, a
// draft a lane), sums its part of the one row that counts, and hands its sum to
// the others; the CTA, and in it the warp, whose part holds the border goes
// through that part again.  Every value is read from memory once, the drafts'
// own probabilities and that last part apart.
#include "b2q_groups.cuh"
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

namespace b2q {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;

// One weight of the draw: target probability p against draft probability q.
// What is not a finite number above 0 counts as 0.
__device__ __forceinline__ double weight(float p, float q) {
  if (!(p > q) || !(p > 0.0f) || p == INFINITY) return 0.0;
  return static_cast<double>(p) - static_cast<double>(q);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyArgs a) {
  using V = typename Val<T>::type;
  __shared__ double sums[kWarps], totals[kVerifyRanks], mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ranks = a.ranks, rank = ranks > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t b = blockIdx.x / ranks;
  const int64_t lo = min(max(static_cast<int64_t>(__ldg(a.cu + b)), int64_t{0}), a.D);
  const int64_t hi = min(max(static_cast<int64_t>(__ldg(a.cu + b + 1)), lo), a.D);
  const V* target = static_cast<const V*>(a.target);
  const V* guess = static_cast<const V*>(a.guess);
  // How many drafts stay: every warp finds out for itself.
  int64_t first = hi;
  for (int64_t i0 = lo; i0 < hi; i0 += 32) {
    const int64_t i = i0 + lane;
    bool keep = true;
    if (i < hi) {
      const int d = __ldg(a.drafts + i);
      keep = false;
      if (d >= 0 && d < a.V) {
        const float p = Val<T>::load(target + (i + b) * a.ldp + d);
        const float q = guess ? Val<T>::load(guess + i * a.ldq + d) : 1.0f;
        keep = static_cast<double>(__ldg(a.u + i)) * static_cast<double>(q) < static_cast<double>(p);
      }
    }
    const unsigned fails = __ballot_sync(0xffffffffu, !keep);
    if (fails) {
      first = i0 + __ffs(fails) - 1;
      break;
    }
  }
  const bool down = first < hi;
  const V* p_row = target + (first + b) * a.ldp;
  const V* q_row = down && guess ? guess + first * a.ldq : nullptr;
  const int skip = down && !guess ? __ldg(a.drafts + first) : -1;  // its draft probability is 1
  if (rank == 0) {
    for (int64_t i = lo + threadIdx.x; i <= hi; i += kThreads)
      if (i != first) a.tokens[i + b] = i < first ? __ldg(a.drafts + i) : -1;
    if (threadIdx.x == 0) a.accepted[b] = static_cast<int32_t>(first - lo);
  }
  // This warp's part of the vocabulary.
  const int64_t part = ((a.V + static_cast<int64_t>(ranks) * kWarps - 1) / (ranks * kWarps) + 31) / 32 * 32;
  const int64_t j0 = min(a.V, (static_cast<int64_t>(rank) * kWarps + warp) * part);
  const int64_t j1 = min(a.V, j0 + part);
  bool residual = down;
  double total = 0.0, before = 0.0;
  while (true) {
    double sum = 0.0;
#pragma unroll 4
    for (int64_t j = j0 + lane; j < j1; j += 32) {
      const float p = Val<T>::load(p_row + j);
      float q = 0.0f;
      if (residual) q = q_row ? Val<T>::load(q_row + j) : (j == skip ? 1.0f : 0.0f);
      sum += weight(p, q);
    }
    sum = warp_sum(sum);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    double cta = 0.0;
    for (int w = 0; w < kWarps; ++w) cta += sums[w];
    if (ranks > 1) {
      if (threadIdx.x == 0) mine = cta;
      cluster_sync();
      if (threadIdx.x < ranks) {
        double v;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr(&mine, threadIdx.x)) : "memory");
        totals[threadIdx.x] = v;
      }
      cluster_sync();  // (and nobody overwrites or leaves before all have read)
    } else {
      if (threadIdx.x == 0) totals[0] = cta;
      __syncthreads();
    }
    total = 0.0, before = 0.0;
    for (int r = 0; r < ranks; ++r) {
      if (r == rank) before = total;
      total += totals[r];
    }
    if (total > 0.0 || !residual) break;
    residual = false;  // nothing is left of p above q
    __syncthreads();
  }
  // The border, and the warp whose part it falls into: the first with a weight
  // whose end lies behind it, or the last with one when rounding (or v >= 1) puts
  // it at the very end.  A CTA's last such warp ends where the next CTA begins,
  // so that the parts meet whatever the sums were rounded to.
  const float v = __ldg(a.v + b);
  const double edge = (v > 0.0f ? static_cast<double>(v) : 0.0) * total;
  int64_t found = -1;
  bool later = false, last_here = true;  // a weight in a later CTA, in a later warp of this one
  double start = before;
  for (int w = 0; w < warp; ++w) start += sums[w];
  for (int w = warp + 1; w < kWarps; ++w) last_here &= sums[w] == 0.0;
  for (int r = rank + 1; r < ranks; ++r) later |= totals[r] > 0.0;
  const double stop = last_here ? before + totals[rank] : start + sums[warp];
  const bool holds = sums[warp] > 0.0 && start <= edge && (edge < stop || (last_here && !later));
  if (total > 0.0) {
    if (holds) {
      double run = start;
      int64_t last = -1;
      for (int64_t jj = j0; jj < j1 && found < 0; jj += 32) {
        const int64_t j = jj + lane;
        double w = 0.0;
        if (j < j1) {
          const float p = Val<T>::load(p_row + j);
          float q = 0.0f;
          if (residual) q = q_row ? Val<T>::load(q_row + j) : (j == skip ? 1.0f : 0.0f);
          w = weight(p, q);
        }
        double inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += up;
        }
        const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && run + inc > edge);
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        if (over) found = jj + __ffs(over) - 1;
        if (some) last = jj + 31 - __clz(some);
        run += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (found < 0) found = last;
      if (lane == 0) a.tokens[first + b] = static_cast<int32_t>(found);
    }
  } else if (rank == 0 && threadIdx.x == 0) {
    a.tokens[first + b] = -1;
  }
}

}  // namespace

cudaError_t launch_verify(VerifyArgs a, int type, cudaStream_t s) {
  a.ranks = kVerifyRanks;
  void (*kernels[3])(const VerifyArgs) = {verify_kernel<0>, verify_kernel<1>, verify_kernel<2>};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(a.ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.B * a.ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernels[type], a);
}

}  // namespace b2q

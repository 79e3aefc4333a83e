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
// draft a lane), sums its part of the one row that counts, a piece a warp, and
// hands its sum to the others.  The CTA that finds the border in the piece of one
// of its warps shares that piece out among all of them again, and so on, until
// what is left is one warp's few values.  Every value is read from memory once,
// those pieces apart.
// Bound by that read; a thread asks for 8 values of each row at a time, and an SM
// has 6 CTAs, so that enough are on their way (rows of any alignment: values are
// read one by one, 32 neighbours a warp).  Measured: 96 requests of up to 7 drafts,
// 151001 tokens, fp32: 27.4 us for 90 MB; 4 requests of 32000 tokens, bf16: 7.8 us (512
// threads a CTA, four values at a time and one warp after the border: 105 and 11).
#include "b2q_groups.cuh"
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

namespace b2q {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRanks = 8;  // CTAs of one request
constexpr int kBatch = 8;  // values of a row that a thread asks for at a time

// One weight of the draw: target probability p above draft probability q (a
// negative q counts as 0).  A p that is not a finite number above 0, or whose q is
// no number, has none.
__device__ __forceinline__ bool counts(float p, float q) { return p > fmaxf(q, 0.0f) && q == q && p < INFINITY; }
__device__ __forceinline__ double weight(float p, float q) {
  return counts(p, q) ? static_cast<double>(p) - static_cast<double>(fmaxf(q, 0.0f)) : 0.0;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int T>
__global__ void __launch_bounds__(kThreads, 6) verify_kernel(const VerifyArgs a) {
  using V = typename Val<T>::type;
  __shared__ double sums[kWarps], totals[kRanks], mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  const int64_t b = blockIdx.x / kRanks;
  grid_wait();
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
    if (b == 0)  // rows before the first request, and behind the last
      for (int64_t i = threadIdx.x; i < lo; i += kThreads) a.tokens[i] = -1;
    if (b == a.B - 1)
      for (int64_t i = hi + 1 + threadIdx.x; i <= a.D; i += kThreads) a.tokens[i + b] = -1;
    if (threadIdx.x == 0) a.accepted[b] = static_cast<int32_t>(first - lo);
  }
  // This warp's part of the vocabulary.
  const int64_t part = ((a.V + kRanks * kWarps - 1) / (kRanks * kWarps) + 31) / 32 * 32;
  const int64_t j0 = min(a.V, (static_cast<int64_t>(rank) * kWarps + warp) * part);
  const int64_t j1 = min(a.V, j0 + part);
  bool residual = down;
  // The weights of the warp's values from j on, 32 a step.
  auto fetch = [&](int64_t j, int64_t end, float (&pv)[kBatch], float (&qv)[kBatch]) {
    const V* pp = p_row + j + lane;
    const V* qq = q_row + j + lane;
    const bool with_q = residual && q_row;
    if (j + kBatch * 32 <= end) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) pv[i] = Val<T>::load(pp + i * 32);
      if (with_q) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) qv[i] = Val<T>::load(qq + i * 32);
        return;
      }
    } else {
      const int left = static_cast<int>(end - j) - lane;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) pv[i] = i * 32 < left ? Val<T>::load(pp + i * 32) : 0.0f;
      if (with_q) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) qv[i] = i * 32 < left ? Val<T>::load(qq + i * 32) : 0.0f;
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) qv[i] = 0.0f;
    if (residual) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) qv[i] = j + i * 32 + lane == skip ? 1.0f : 0.0f;
    }
  };
  auto sum_of = [&](int64_t from, int64_t end) {
    // (One conversion to 64 bits a weight instead of two: the difference, and in `rest` what rounding it to 32 left,
    // which is exact; the sum of those needs no more than 32 bits.)
    double sum = 0.0;
    float rest = 0.0f;
    for (int64_t j = from; j < end; j += kBatch * 32) {
      float pv[kBatch], qv[kBatch];
      fetch(j, end, pv, qv);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float q = fmaxf(qv[i], 0.0f);
        const bool in = counts(pv[i], qv[i]);
        const float d = in ? pv[i] - q : 0.0f;
        sum += static_cast<double>(d);
        rest += in ? (pv[i] - d) - q : 0.0f;
      }
    }
    return warp_sum(sum + static_cast<double>(rest));
  };
  double total = 0.0, before = 0.0;
  while (true) {
    const double sum = sum_of(j0, j1);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    double cta = 0.0;
    for (int w = 0; w < kWarps; ++w) cta += sums[w];
    if (threadIdx.x == 0) mine = cta;
    cluster_sync();
    if (threadIdx.x < kRanks) {
      double v;
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr(&mine, threadIdx.x)) : "memory");
      totals[threadIdx.x] = v;
    }
    cluster_sync();  // (and nobody overwrites or leaves before all have read)
    total = 0.0, before = 0.0;
    for (int r = 0; r < kRanks; ++r) {
      if (r == rank) before = total;
      total += totals[r];
    }
    if (total > 0.0 || !residual) break;
    residual = false;  // nothing is left of p above q
    __syncthreads();
  }
  if (total > 0.0) {
    // The border, and the piece it falls into: the first with a weight whose end lies
    // behind it, or the last with one when rounding (or v >= 1) puts it at the
    // very end.  The last such piece of what is shared out ends where that ends, so
    // that pieces meet whatever their sums were rounded to.
    const float v = __ldg(a.v + b);
    const double edge = (v > 0.0f ? static_cast<double>(v) : 0.0) * total;
    bool later = false;  // a weight behind what is shared out
    for (int r = rank + 1; r < kRanks; ++r) later |= totals[r] > 0.0;
    double start = before, stop = before + totals[rank];
    int64_t from = static_cast<int64_t>(rank) * kWarps * part, size = part;
    bool here = totals[rank] > 0.0 && start <= edge && (edge < stop || !later);
    while (here) {  // (the same in all threads of the CTA)
      int holder = -1;
      double run = start, begin = start, end = start;
      bool after = later;
      for (int w = 0; w < kWarps; ++w) {
        if (sums[w] == 0.0) continue;
        // the last one with a weight so far; an earlier one holds the border if it ends behind it
        if (holder >= 0 && edge < end) {
          after = true;
          break;
        }
        holder = w;
        begin = run;
        run += sums[w];
        end = run;
      }
      if (holder < 0) break;  // (sums that are not 0 had such a piece)
      bool last = true;
      for (int w = holder + 1; w < kWarps; ++w) last &= sums[w] == 0.0;
      if (last) end = stop;
      later = after || !last || later;
      start = begin;
      stop = end;
      const int64_t limit = min(a.V, from + (holder + 1) * size);
      from += holder * size;
      if (size <= 2 * kBatch * 32) {
        if (warp != holder) break;
        double sum = start;
        int64_t found = -1, seen = -1;
        for (int64_t j = from; j < limit && found < 0; j += kBatch * 32) {
          float pv[kBatch], qv[kBatch];
          fetch(j, limit, pv, qv);
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const double w = weight(pv[i], qv[i]);
            double inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double up = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += up;
            }
            const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && sum + inc > edge);
            const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
            if (over && found < 0) found = j + i * 32 + __ffs(over) - 1;
            if (some && found < 0) seen = j + i * 32 + 31 - __clz(some);
            sum += __shfl_sync(0xffffffffu, inc, 31);
          }
        }
        if (lane == 0) a.tokens[first + b] = static_cast<int32_t>(found >= 0 ? found : seen);
        break;
      }
      // Share the piece out again.
      size = ((limit - from + kWarps - 1) / kWarps + 31) / 32 * 32;
      const double sum = sum_of(from + warp * size, min(limit, from + (warp + 1) * size));
      __syncthreads();  // the sums before are no longer read
      if (lane == 0) sums[warp] = sum;
      __syncthreads();
    }
  } else if (rank == 0 && threadIdx.x == 0) {
    a.tokens[first + b] = -1;
  }
}

}  // namespace

cudaError_t launch_verify(const VerifyArgs& a, int type, cudaStream_t s) {
  void (*kernels[3])(const VerifyArgs) = {verify_kernel<0>, verify_kernel<1>, verify_kernel<2>};
  return launch_early(kernels[type], dim3(static_cast<unsigned>(a.B * kRanks)), dim3(kThreads), 0, s, kRanks, a);
}

}  // namespace b2q

// b2q_mul_mat_id.cu -- matrix products whose weight goes by row: slot s of a
// plan multiplies the weight of its expert,
//   y[s][r] = sum_k W[e(s)][r][k] x[s / per_row][k] (+ bias[e][r]),
// or, with GLU, silu(y[s][r]) * y[s][n + r] of a weight of 2 n rows.
//
// Plain form: a CTA has one tile of 32 sorted slots and 64 weight rows, staged
// in shared memory as fp32, 32 of K at a time.
#include "b2q_groups.cuh"
#include "b2q_internal.h"

namespace b2q {

namespace {

constexpr int kSlots = 32, kRows = 64, kDepth = 32, kThreads = 256;

template <int W>
__device__ __forceinline__ float weight_at(const MulMatIdArgs& a, int e, int64_t row, int64_t k) {
  if constexpr (W == 3) {  // Q4_0: nibbles [E * rows][K / 2], scales fp16 [K / 32][lds]
    const int64_t r = static_cast<int64_t>(e) * a.rows + row;
    const uint8_t b = static_cast<const uint8_t*>(a.w)[r * (a.K / 2) + (k / 32) * 16 + (k % 16)];
    const int q = (k % 32) < 16 ? (b & 15) : (b >> 4);
    const __half d = reinterpret_cast<const __half*>(a.scales)[(k / 32) * a.lds + r];
    return __half2float(d) * static_cast<float>(q - 8);
  } else {
    using V = typename Val<W>::type;
    return Val<W>::load(static_cast<const V*>(a.w) + e * a.expert_stride + row * a.ldw + k);
  }
}

template <int W, int X, int Y>
__global__ void __launch_bounds__(kThreads) mul_mat_id_kernel(const MulMatIdArgs a) {
  using XV = typename Val<X>::type;
  using YV = typename Val<Y>::type;
  __shared__ float xs[kSlots][kDepth + 1], ws[2][kRows][kDepth + 1];
  __shared__ int slot[kSlots];
  const GroupTile t = find_group_tile(a.offsets, a.E, a.S, blockIdx.x, kSlots);
  if (t.group < 0) return;
  const int count = t.end - t.begin;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kRows;
  if (threadIdx.x < kSlots) {
    int s = -1;
    if (static_cast<int>(threadIdx.x) < count) {
      s = __ldg(a.order + t.begin + threadIdx.x);
      if (s < 0 || s >= a.S) s = -1;
    }
    slot[threadIdx.x] = s;
  }
  __syncthreads();
  const int row = threadIdx.x % kRows, part = threadIdx.x / kRows;  // 4 parts of 8 slots
  float acc[2][8] = {};
  if (t.group < a.E) {
    const int halves = a.glu ? 2 : 1;
    for (int64_t k0 = 0; k0 < a.K; k0 += kDepth) {
      for (int i = threadIdx.x; i < kSlots * kDepth; i += kThreads) {
        const int m = i / kDepth, k = i % kDepth;
        float v = 0.0f;
        if (slot[m] >= 0 && k0 + k < a.K)
          v = Val<X>::load(static_cast<const XV*>(a.x) + (slot[m] / a.per_row) * a.ldx + k0 + k);
        xs[m][k] = v;
      }
      for (int h = 0; h < halves; ++h)
        for (int i = threadIdx.x; i < kRows * kDepth; i += kThreads) {
          const int r = i / kDepth, k = i % kDepth;
          ws[h][r][k] = r0 + r < a.n && k0 + k < a.K ? weight_at<W>(a, t.group, h * a.n + r0 + r, k0 + k) : 0.0f;
        }
      __syncthreads();
      for (int h = 0; h < halves; ++h)
        for (int k = 0; k < kDepth; ++k) {
          const float w = ws[h][row][k];
#pragma unroll
          for (int m = 0; m < 8; ++m) acc[h][m] = fmaf(w, xs[part * 8 + m][k], acc[h][m]);
        }
      __syncthreads();
    }
  }
  if (r0 + row >= a.n) return;
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    const int s = slot[part * 8 + m];
    if (s < 0) continue;
    float v = 0.0f;
    if (t.group < a.E) {
      const float* b = a.bias ? a.bias + t.group * a.rows + r0 + row : nullptr;
      v = acc[0][m] + (b ? b[0] : 0.0f);
      if (a.glu) v = v / (1.0f + expf(-v)) * (acc[1][m] + (b ? b[a.n] : 0.0f));
    }
    static_cast<YV*>(a.y)[s * a.ldy + r0 + row] = Val<Y>::to(v);
  }
}

}  // namespace

cudaError_t launch_mul_mat_id(const MulMatIdArgs& a, int wtype, int xtype, int ytype, cudaStream_t s) {
  void (*k)(const MulMatIdArgs) = nullptr;
  if (wtype == 1) k = ytype == 0 ? mul_mat_id_kernel<1, 1, 0> : mul_mat_id_kernel<1, 1, 1>;
  if (wtype == 2) k = ytype == 0 ? mul_mat_id_kernel<2, 2, 0> : mul_mat_id_kernel<2, 2, 2>;
  if (wtype == 3) k = ytype == 0 ? mul_mat_id_kernel<3, 1, 0> : mul_mat_id_kernel<3, 1, 1>;
  if (!k) return cudaErrorInvalidValue;
  (void)xtype;
  const int64_t tiles = a.S / kSlots + a.E + 1;
  k<<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>((a.n + kRows - 1) / kRows)), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace b2q

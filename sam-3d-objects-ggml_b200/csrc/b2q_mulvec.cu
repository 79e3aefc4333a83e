// b2q_mulvec.cu -- products of at most kMulVecMaxM tokens with a 4-bit weight
// whose values are taken as they stand (no 8-bit rounding of the activations):
//   Q4_0 (compact layout)  y[m][n] = sum_b d[n,b] sum_i (q_i - 8) x[m][i]
//   Q4_K (GGUF rows)       y[m][n] = sum_s d sc_s sum_i q_i x[m][i] - dmin mn_s sum_i x[m][i]
// then bias, gate and residual as the other few-token product has them.
// One warp per weight row, lanes over the 32-value blocks, fp32 throughout.
#include "b2q_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2q {

namespace {

constexpr int kMvThreads = 256;

template <int XT>
__device__ __forceinline__ float x_at(const void* x, int64_t i) {
  if constexpr (XT == kXF32) return __ldg(static_cast<const float*>(x) + i);
  if constexpr (XT == kXF16) return __half2float(__ldg(static_cast<const __half*>(x) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(x) + i));
}

template <bool Q4K, int XT>
__global__ void __launch_bounds__(kMvThreads) mul_vec_kernel(const MulVecArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kMvThreads / 32) + (threadIdx.x >> 5);
  if (n >= a.N) return;
  float acc[kMulVecMaxM] = {};
  for (int64_t b = lane; b < a.K / 32; b += 32) {
    float d, off;
    uint32_t q[4];  // 8 codes each
    if constexpr (Q4K) {
      const uint8_t* blk = a.w + n * a.row_bytes + (b / 8) * kQ4KBytes;
      const int j = static_cast<int>(b % 8);
      const float fd = __half2float(*reinterpret_cast<const __half*>(blk));
      const float fm = __half2float(*reinterpret_cast<const __half*>(blk + 2));
      const uint8_t* sc = blk + 4;
      const int scale = j < 4 ? sc[j] & 63 : (sc[j + 4] & 15) | ((sc[j - 4] >> 6) << 4);
      const int mn = j < 4 ? sc[j + 4] & 63 : (sc[j + 4] >> 4) | ((sc[j] >> 6) << 4);
      d = fd * static_cast<float>(scale);
      off = -fm * static_cast<float>(mn);
      const uint32_t* c = reinterpret_cast<const uint32_t*>(blk + 16 + 32 * (j / 2));
      for (int m = 0; m < a.M; ++m) {
        float s = 0.0f, sx = 0.0f;
        for (int i = 0; i < 32; ++i) {
          const float x = x_at<XT>(a.x, m * a.ldx + b * 32 + i);
          s = fmaf(static_cast<float>((c[i / 4] >> (8 * (i % 4) + 4 * (j & 1))) & 15), x, s);
          sx += x;
        }
        acc[m] = fmaf(d, s, fmaf(off, sx, acc[m]));
      }
    } else {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(a.w + n * (a.K / 2) + b * 16));
      q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w;
      d = __half2float(__ushort_as_half(a.scales[b * a.lds + n]));
      for (int m = 0; m < a.M; ++m) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int code = (q[(i % 16) / 4] >> (8 * (i % 4) + (i / 16) * 4)) & 15;
          s = fmaf(static_cast<float>(code - 8), x_at<XT>(a.x, m * a.ldx + b * 32 + i), s);
        }
        acc[m] = fmaf(d, s, acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kMulVecMaxM; ++m) {
    float v = acc[m];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane != 0 || m >= a.M) continue;
    if (a.bias) v = __fadd_rn(v, a.bias[n]);
    if (a.resid) v = __fadd_rn(a.resid[m * a.ldr + n], a.gate ? __fmul_rn(v, a.gate[n]) : v);
    a.y[m * a.ldy + n] = v;
  }
}

}  // namespace

cudaError_t launch_mul_vec(const MulVecArgs& a, bool q4k, int xt, int num_sms, cudaStream_t s) {
  (void)num_sms;
  const int64_t grid = (a.N + kMvThreads / 32 - 1) / (kMvThreads / 32);
  const unsigned g = static_cast<unsigned>(grid);
#define B2Q_MV(Q, X) mul_vec_kernel<Q, X><<<g, kMvThreads, 0, s>>>(a)
  if (q4k) {
    if (xt == kXF32) B2Q_MV(true, kXF32); else if (xt == kXF16) B2Q_MV(true, kXF16); else B2Q_MV(true, kXBF16);
  } else {
    if (xt == kXF32) B2Q_MV(false, kXF32); else if (xt == kXF16) B2Q_MV(false, kXF16); else B2Q_MV(false, kXBF16);
  }
#undef B2Q_MV
  return cudaGetLastError();
}

}  // namespace b2q

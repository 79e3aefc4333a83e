// b2q_rope.cu -- fused qkv rows to a cached attention's inputs: per-head RMS
// norm of q and k, rotary positions with up to three axes, q rows out and k, v
// appended to the paged cache, in one pass.
//
//   h' = h * gamma / sqrt(mean(h^2) + eps)                    (norm, q and k)
//   pair i (dims (i, i + R), or (2i, 2i + 1) interleaved), axis x(i), i < R:
//     angle = pos[x(i)][t] * f_i,  (a, b) -> (a cos - b sin, b cos + a sin)
//   k, v of token t to slot[t] of [page][kv head][token in page][D]
//
// Bound by its bytes: 4 read and 2 written per value of a row, each once.  A
// CTA takes kRopeTokens (or one, where there are few) tokens: its threads
// first compute the tokens' cosines and sines into shared memory, one pair
// each, which all the heads then share; a row of D values is D / 4 lanes of
// one float4 each, so a warp's access is 512 contiguous bytes, and the RMS
// sum and the partner of a pair are shuffles inside that group of lanes.
//
// The angle is formed in double and reduced to a fraction of a turn before it
// is rounded to fp32: in fp32 the product of a position of 10^4 and a frequency
// near 1 would already be 5e-4 radians off, half an fp16 ulp of the result.
#include "b2q_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2q {

namespace {

constexpr int kRopeThreads = 256;

template <bool BF16>
__device__ __forceinline__ uint2 pack4(float4 v) {
  uint2 r;
  if constexpr (BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    r.x = *reinterpret_cast<const uint32_t*>(&a);
    r.y = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    r.x = *reinterpret_cast<const uint32_t*>(&a);
    r.y = *reinterpret_cast<const uint32_t*>(&b);
  }
  return r;
}

// sum over the LPR lanes of a row
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kRopeThreads) rope_cache_kernel(const RopeArgs a, int tokens_per_cta) {
  constexpr int LPR = D / 4;            // lanes per row
  constexpr int RPP = kRopeThreads / LPR;  // rows per pass of the CTA
  extern __shared__ float2 rope_cs[];   // [tokens_per_cta][R] (cos, sin)
  const int tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_cta;
  const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_cta), a.T - t0));
  const int R = a.rot;
  for (int i = tid; i < nt * R; i += kRopeThreads) {
    const int t = i / R, p = i - t * R;
    const int axis = p >= a.sec1 ? (p >= a.sec2 ? 2 : 1) : 0;
    const double turns = static_cast<double>(a.pos[axis * a.ldpos + t0 + t]) *
                         (static_cast<double>(a.inv_freq[p]) * 0.15915494309189535);  // 1 / (2 pi)
    float sn, cs;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
    rope_cs[i] = make_float2(cs, sn);
  }
  __syncthreads();

  const int heads = a.Hq + 2 * a.Hkv;
  const int h_lo = static_cast<int>(static_cast<int64_t>(heads) * blockIdx.y / gridDim.y);
  const int h_n = static_cast<int>(static_cast<int64_t>(heads) * (blockIdx.y + 1) / gridDim.y) - h_lo;
  const int l = tid % LPR, r0 = tid / LPR;
  const int n_rows = nt * h_n;
  const unsigned group = (LPR == 32) ? 0 : (tid & 31) / LPR * LPR;  // first lane of this row's group
  // Every lane runs every pass (the shuffles name the whole warp); rows past
  // the end reload the last row and store nothing.
  for (int r = r0; r - r0 < n_rows; r += RPP) {
    const int rc = min(r, n_rows - 1);
    const int tl = rc / h_n, h = h_lo + (rc - tl * h_n);
    const int64_t t = t0 + tl;
    const float* row = a.qkv + t * a.ldqkv + static_cast<int64_t>(h) * D;
    float4 v = __ldg(reinterpret_cast<const float4*>(row) + l);
    const bool is_v = h >= a.Hq + a.Hkv;
    // (the shuffles below run for v rows too: a warp may hold both kinds)
    float scale = 1.0f;
    if (a.norm) {
      const float ss = row_sum<LPR>((v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w));
      if (!is_v) scale = rsqrtf(ss * (1.0f / D) + a.eps);
    }
    const float* gamma = is_v ? nullptr : (h < a.Hq ? a.gamma_q : a.gamma_k);
    const int64_t g0 = static_cast<int64_t>(h < a.Hq ? h : h - a.Hq) * D;
    if (a.norm && !is_v) {
      v.x *= scale, v.y *= scale, v.z *= scale, v.w *= scale;
      if (gamma) {
        const float4 g = __ldg(reinterpret_cast<const float4*>(gamma + g0) + l);
        v.x *= g.x, v.y *= g.y, v.z *= g.z, v.w *= g.w;
      }
    }
    const int d0 = 4 * l;
    const float2* cs = rope_cs + tl * R;
    if (a.interleaved) {
      if (!is_v) {
        if (d0 < 2 * R) {
          const float2 c = cs[2 * l];
          const float x = v.x * c.x - v.y * c.y;
          v.y = v.y * c.x + v.x * c.y;
          v.x = x;
        }
        if (d0 + 2 < 2 * R) {
          const float2 c = cs[2 * l + 1];
          const float x = v.z * c.x - v.w * c.y;
          v.w = v.w * c.x + v.z * c.y;
          v.z = x;
        }
      }
    } else if (R % 4 == 0) {  // the four partners sit in one lane
      const bool second = d0 >= R;
      const int src = static_cast<int>(group) + (second ? (l - R / 4 + LPR) % LPR : (l + R / 4) % LPR);
      float4 o;
      o.x = __shfl_sync(0xffffffffu, v.x, src);
      o.y = __shfl_sync(0xffffffffu, v.y, src);
      o.z = __shfl_sync(0xffffffffu, v.z, src);
      o.w = __shfl_sync(0xffffffffu, v.w, src);
      if (!is_v && d0 < 2 * R) {
        const float4* c4 = reinterpret_cast<const float4*>(cs + (second ? d0 - R : d0));
        const float4 c01 = c4[0], c23 = c4[1];
        const float sg = second ? 1.0f : -1.0f;
        v.x = v.x * c01.x + sg * (o.x * c01.y);
        v.y = v.y * c01.z + sg * (o.y * c01.w);
        v.z = v.z * c23.x + sg * (o.z * c23.y);
        v.w = v.w * c23.z + sg * (o.w * c23.w);
      }
    } else if (!is_v) {  // partners across lanes: read them from the row itself
      float* e = reinterpret_cast<float*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d0 + i;
        if (d >= 2 * R) continue;
        const bool second = d >= R;
        const int dp = second ? d - R : d + R;
        float o = __ldg(row + dp) * scale;
        if (a.norm && gamma) o *= __ldg(gamma + g0 + dp);
        const float2 c = cs[second ? dp : d];
        e[i] = e[i] * c.x + (second ? o * c.y : -(o * c.y));
      }
    }
    if (r >= n_rows) continue;
    const uint2 w = pack4<BF16>(v);
    if (h < a.Hq) {
      *(reinterpret_cast<uint2*>(a.q + t * a.ldq + static_cast<int64_t>(h) * D) + l) = w;
    } else {
      const int64_t slot = a.slots[t];
      if (slot >= 0 && slot < a.n_slots) {
        const int hk = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
        const int64_t page = slot >> a.page_shift, off = slot & ((int64_t{1} << a.page_shift) - 1);
        uint16_t* cache = is_v ? a.v_cache : a.k_cache;
        *(reinterpret_cast<uint2*>(cache + ((((page * a.Hkv + hk) << a.page_shift) + off) * D)) + l) = w;
      }
    }
  }
}

}  // namespace

cudaError_t launch_rope_cache(const RopeArgs& a, int D, bool bf16, int num_sms, cudaStream_t s) {
  const int heads = a.Hq + 2 * a.Hkv;
  const int rows_per_pass = kRopeThreads / (D / 4);
  // Tokens per CTA: as many as fill the threads with one pair each, while that
  // still gives every SM two CTAs; with fewer tokens, one per CTA and the heads
  // shared out over grid.y, down to one pass of rows each.
  int tpc = a.rot > 0 ? kRopeThreads / a.rot : kRopeThreads / (D / 2);
  if (tpc > 8) tpc = 8;
  if (a.T < static_cast<int64_t>(tpc) * num_sms * 2) tpc = 1;
  const int64_t gx = (a.T + tpc - 1) / tpc;
  if (gx > INT32_MAX) return cudaErrorInvalidValue;
  int64_t gy = 1;
  if (tpc == 1 && gx < 2 * num_sms) {
    gy = (2 * num_sms + gx - 1) / gx;
    const int64_t most = (heads + rows_per_pass - 1) / rows_per_pass;
    if (gy > most) gy = most;
  }
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  const int smem = tpc * (a.rot > 0 ? a.rot : 1) * 8;
#define B2Q_ROPE(DD, BF) rope_cache_kernel<DD, BF><<<grid, kRopeThreads, smem, s>>>(a, tpc)
  if (D == 64) {
    if (bf16) B2Q_ROPE(64, true); else B2Q_ROPE(64, false);
  } else {
    if (bf16) B2Q_ROPE(128, true); else B2Q_ROPE(128, false);
  }
#undef B2Q_ROPE
  return cudaGetLastError();
}

}  // namespace b2q

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
// CTA takes up to kRopeTokens tokens (one, where there are few): its threads
// first compute the tokens' cosines and sines into shared memory, one pair
// each, which all the heads then share.  A lane takes 8 values that hold whole pairs (8 neighbours, or for pairs
// (i, i + R) four neighbours and their four partners), so a head is D / 8 lanes
// and the RMS sum is shuffles among them; a thread's next rows are loaded while it
// works on these.  q and k rows and v rows are two loops, and the kinds of rotation
// and norm are template arguments: with one loop of 4-value lanes the rows cost 136
// instructions a warp, and 32800 tokens of 48 heads of 64 took 200 us where this
// takes 102 (5950 GB/s).  With pairs (i, i + R) and 40 heads of 128: 160 us, 6290
// GB/s, and 207 when the partners came by shuffles.  24 tokens of 40 heads of 128:
// 3.2 us, a launch and one round of loads and stores.
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
constexpr int kRopeTokens = 8;  // most tokens of a CTA
constexpr int kRopeBatch = 2;   // rows of a thread whose loads are under way together
enum { kInterleaved = 0, kHalves = 1, kHalvesOdd = 2 };  // pairs (2i, 2i + 1); (i, i + R), R % 4 == 0; any R

struct F8 {
  float v[8];
};
__device__ __forceinline__ F8 load8(const float* p) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
// four values and four more
__device__ __forceinline__ F8 load44(const float* p, const float* q) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(q));
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const F8& f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const __nv_bfloat162 x = __floats2bfloat162_rn(f.v[2 * i], f.v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&x);
    } else {
      const __half2 x = __floats2half2_rn(f.v[2 * i], f.v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// 16 bytes to a row that is 8-byte aligned at least
__device__ __forceinline__ void store8(uint16_t* dst, uint4 w, bool wide) {
  if (wide) {
    __stcs(reinterpret_cast<uint4*>(dst), w);
  } else {
    __stcs(reinterpret_cast<uint2*>(dst), make_uint2(w.x, w.y));
    __stcs(reinterpret_cast<uint2*>(dst) + 1, make_uint2(w.z, w.w));
  }
}

// sum over the LPR lanes of a row
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A thread's rows (token, head) of n heads, `step` rows apart.
struct RowWalk {
  int tl, h, n, dt, dh;
  __device__ __forceinline__ RowWalk(int first, int step, int heads) : n(heads) {
    tl = first / n;
    h = first - tl * n;
    dt = step / n;
    dh = step - dt * n;
  }
  __device__ __forceinline__ void next() {
    tl += dt;
    h += dh;
    if (h >= n) h -= n, ++tl;
  }
};

// (four CTAs an SM: with registers for fewer the 32800 tokens above take 112 us, for five 109)
template <int D, bool BF16, bool NORM, int MODE>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_cache_kernel(const RopeArgs a, int tokens_per_cta, bool wide) {
  constexpr int LPR = D / 8;               // lanes per row
  constexpr int RPP = kRopeThreads / LPR;  // rows per pass of the CTA
  extern __shared__ __align__(16) float2 rope_cs[];  // [tokens_per_cta][R] (cos, sin)
  __shared__ int64_t rope_at[kRopeTokens];           // a token's place in kv head 0 of the cache, or -1
  const int tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_cta;
  const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_cta), a.T - t0));
  const int R = a.rot;
  // this CTA's heads: lo .. hi - 1 of q, k, v heads in a row
  const int heads = a.Hq + 2 * a.Hkv, n_qk = a.Hq + a.Hkv;
  const int lo = static_cast<int>(static_cast<int64_t>(heads) * blockIdx.y / gridDim.y);
  const int hi = static_cast<int>(static_cast<int64_t>(heads) * (blockIdx.y + 1) / gridDim.y);
  const int l = tid % LPR;
  for (int i = tid; i < nt * R; i += kRopeThreads) {
    const int t = i / R, p = i - t * R;
    const int axis = p >= a.sec1 ? (p >= a.sec2 ? 2 : 1) : 0;
    const double turns = static_cast<double>(a.pos[axis * a.ldpos + t0 + t]) *
                         (static_cast<double>(a.inv_freq[p]) * 0.15915494309189535);  // 1 / (2 pi)
    float sn, cs;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
    rope_cs[i] = make_float2(cs, sn);
  }
  if (tid < nt && a.Hkv > 0) {
    const int64_t slot = a.slots[t0 + tid];
    const int64_t page = slot >> a.page_shift, off = slot & ((int64_t{1} << a.page_shift) - 1);
    rope_at[tid] = slot >= 0 && slot < a.n_slots ? ((page * a.Hkv << a.page_shift) + off) * D : -1;
  }
  __syncthreads();
  const int64_t head_step = static_cast<int64_t>(D) << a.page_shift;

  // Every lane runs every pass (the shuffles name the whole warp); rows past the
  // end repeat the CTA's last token and store nothing.
  if (lo < min(hi, n_qk)) {
    const int n = min(hi, n_qk) - lo, rows = nt * n;
    RowWalk w(tid / LPR, RPP, n);
    // A lane's values: four from da and four from db, neighbours but for pairs of halves,
    // where the second four are the partners of the first (past the pairs, neighbours again).
    int da = 8 * l, db = 8 * l + 4;
    if (MODE == kHalves && 4 * l < R) da = 4 * l, db = R + 4 * l;
    for (int r = 0; r < rows; r += kRopeBatch * RPP) {
      F8 x[kRopeBatch];
      int xt[kRopeBatch], xh[kRopeBatch];
      float scale[kRopeBatch];
#pragma unroll
      for (int u = 0; u < kRopeBatch; ++u) {
        xt[u] = w.tl;
        xh[u] = lo + w.h;
        const float* row = a.qkv + (t0 + min(w.tl, nt - 1)) * a.ldqkv + static_cast<int64_t>(xh[u]) * D;
        x[u] = load44(row + da, row + db);
        w.next();
      }
      if constexpr (NORM) {
#pragma unroll
        for (int u = 0; u < kRopeBatch; ++u) {
          float ss = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = fmaf(x[u].v[i], x[u].v[i], ss);
          scale[u] = ss;
        }
#pragma unroll
        for (int u = 0; u < kRopeBatch; ++u) scale[u] = rsqrtf(row_sum<LPR>(scale[u]) * (1.0f / D) + a.eps);
      }
#pragma unroll
      for (int u = 0; u < kRopeBatch; ++u) {
        const int h = xh[u], tt = min(xt[u], nt - 1);
        const float* gamma = h < a.Hq ? a.gamma_q : a.gamma_k;
        const int64_t g0 = static_cast<int64_t>(h < a.Hq ? h : h - a.Hq) * D;
        F8& v = x[u];
        if constexpr (NORM) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v.v[i] *= scale[u];
          if (gamma) {
            const F8 g = load44(gamma + g0 + da, gamma + g0 + db);
#pragma unroll
            for (int i = 0; i < 8; ++i) v.v[i] *= g.v[i];
          }
        }
        const float2* cs = rope_cs + tt * R;
        if constexpr (MODE == kInterleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * l + i < R) {
              const float2 c = cs[4 * l + i];
              const float y = v.v[2 * i] * c.x - v.v[2 * i + 1] * c.y;
              v.v[2 * i + 1] = v.v[2 * i + 1] * c.x + v.v[2 * i] * c.y;
              v.v[2 * i] = y;
            }
        } else if constexpr (MODE == kHalves) {
          if (4 * l < R) {
            const float4* c4 = reinterpret_cast<const float4*>(cs + 4 * l);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float4 c = c4[i];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float x0 = v.v[2 * i + k], x1 = v.v[4 + 2 * i + k], cc = k ? c.z : c.x, sn = k ? c.w : c.y;
                v.v[2 * i + k] = x0 * cc - x1 * sn;
                v.v[4 + 2 * i + k] = x1 * cc + x0 * sn;
              }
            }
          }
        } else {  // partners across lanes: read them from the row itself
          const float* row = a.qkv + (t0 + tt) * a.ldqkv + static_cast<int64_t>(h) * D;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = 8 * l + i;
            if (d >= 2 * R) continue;
            const bool second = d >= R;
            const int dp = second ? d - R : d + R;
            float o = __ldg(row + dp);
            if constexpr (NORM) {
              o *= scale[u];
              if (gamma) o *= __ldg(gamma + g0 + dp);
            }
            const float2 c = cs[second ? dp : d];
            v.v[i] = v.v[i] * c.x + (second ? o * c.y : -(o * c.y));
          }
        }
        if (xt[u] >= nt) continue;
        const uint4 p = pack8<BF16>(v);
        const auto put = [&](uint16_t* row) {
          if constexpr (MODE == kHalves) {
            __stcs(reinterpret_cast<uint2*>(row + da), make_uint2(p.x, p.y));
            __stcs(reinterpret_cast<uint2*>(row + db), make_uint2(p.z, p.w));
          } else {
            store8(row + 8 * l, p, wide);
          }
        };
        if (h < a.Hq) {
          put(a.q + (t0 + tt) * a.ldq + static_cast<int64_t>(h) * D);
        } else {
          const int64_t at = rope_at[tt];
          if (at >= 0) put(a.k_cache + at + (h - a.Hq) * head_step);
        }
      }
    }
  }
  if (max(lo, n_qk) < hi) {
    const int h0 = max(lo, n_qk), n = hi - h0, rows = nt * n;
    RowWalk w(tid / LPR, RPP, n);
    for (int r = 0; r < rows; r += 2 * kRopeBatch * RPP) {
      F8 x[2 * kRopeBatch];
      int xt[2 * kRopeBatch], xh[2 * kRopeBatch];
#pragma unroll
      for (int u = 0; u < 2 * kRopeBatch; ++u) {
        xt[u] = w.tl;
        xh[u] = h0 + w.h;
        if (w.tl < nt) x[u] = load8(a.qkv + (t0 + w.tl) * a.ldqkv + static_cast<int64_t>(xh[u]) * D + 8 * l);
        w.next();
      }
#pragma unroll
      for (int u = 0; u < 2 * kRopeBatch; ++u) {
        if (xt[u] >= nt) continue;
        const int64_t at = rope_at[xt[u]];
        if (at >= 0) store8(a.v_cache + at + (xh[u] - n_qk) * head_step + 8 * l, pack8<BF16>(x[u]), wide);
      }
    }
  }
}

}  // namespace

cudaError_t launch_rope_cache(const RopeArgs& a, int D, bool bf16, int num_sms, cudaStream_t s) {
  const int heads = a.Hq + 2 * a.Hkv;
  const int rows_per_pass = kRopeThreads / (D / 8);
  // Tokens per CTA: as many as fill the threads with one pair each, while that
  // still gives every SM two CTAs; with fewer tokens, one per CTA and the heads
  // shared out over grid.y, down to one pass of rows each.
  int tpc = a.rot > 0 ? kRopeThreads / a.rot : kRopeThreads / (D / 2);
  if (tpc > kRopeTokens) tpc = kRopeTokens;
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
  const auto odd = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  const bool wide = !odd(a.q) && a.ldq % 8 == 0 && !odd(a.k_cache) && !odd(a.v_cache);
  const int mode = a.interleaved ? kInterleaved : a.rot % 4 == 0 ? kHalves : kHalvesOdd;
#define B2Q_ROPE(DD, BF, NO, MO) rope_cache_kernel<DD, BF, NO, MO><<<grid, kRopeThreads, smem, s>>>(a, tpc, wide)
#define B2Q_ROPE_M(DD, BF, NO)                                        \
  do {                                                                \
    if (mode == kInterleaved) B2Q_ROPE(DD, BF, NO, kInterleaved);     \
    else if (mode == kHalves) B2Q_ROPE(DD, BF, NO, kHalves);          \
    else B2Q_ROPE(DD, BF, NO, kHalvesOdd);                            \
  } while (0)
#define B2Q_ROPE_N(DD, BF)                 \
  do {                                     \
    if (a.norm) B2Q_ROPE_M(DD, BF, true);  \
    else B2Q_ROPE_M(DD, BF, false);        \
  } while (0)
  if (D == 64) {
    if (bf16) B2Q_ROPE_N(64, true); else B2Q_ROPE_N(64, false);
  } else {
    if (bf16) B2Q_ROPE_N(128, true); else B2Q_ROPE_N(128, false);
  }
#undef B2Q_ROPE_N
#undef B2Q_ROPE_M
#undef B2Q_ROPE
  return cudaGetLastError();
}

}  // namespace b2q

// b2q_lora.cu -- low-rank adapters of many requests beside a shared projection:
//   y[t] = resid[t] + scale_g * B_g (A_g x[t]),  g = the adapter of row t
// (rows of no adapter: y[t] = resid[t]).
//
// Bound by the rows' bytes (x read, resid read, y written) or, for single tokens,
// by latency.  One launch: a cluster of 8 CTAs has a tile of 16 or 64 sorted rows.
//   1  each CTA multiplies its eighth of K: h = A x, m16n8k16 products
//   2  the partial h meet in the CTAs' shared memories: each CTA adds up the eighth
//      of the rows that is its own, scales them, and hands them to all eight
//   3  each CTA makes its eighth of the columns of y
// so x, resid and y are moved once and no partial result leaves the chip.  h enters
// the second product as two 16-bit numbers (the value and what rounding it left)
// of a power of two per row, so neither fp16's range nor 8 bits of bf16 limit it.
// K and the rank are taken in an order that suits the loads: lane q of a quad has
// 8 consecutive values of every 32 (4 of 16 where the rank is at most 16).
#include "b2q_groups.cuh"
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

#include <algorithm>

namespace b2q {

namespace {

constexpr int kRanks = 8;  // CTAs of a cluster
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kStageK = 64;

template <int MT, int RP>  // 16-row groups of a tile; rank, padded to 16, 32, 64 or 128
struct LoraShape {
  static constexpr int M = 16 * MT;
  static constexpr int SPLIT = kWarps / MT;  // warps that share a row group's K
  static constexpr int PIPE = MT == 1 ? 0 : kStages * (M + RP) * 128;
  static constexpr int PART = kWarps * 16 * RP * 4;
  static constexpr int SUM = M * RP * 4;     // this CTA's h
  static constexpr int PITCH = RP * 2 + (RP >= 64 ? 64 : 0);  // bytes of a row of h's 16-bit numbers: conflict-free reads
  static constexpr int OFF_SUM = PART;
  static constexpr int OFF_H = (PIPE > PART + SUM ? PIPE : PART + SUM);
  static constexpr int OFF_EXP = OFF_H + 2 * M * PITCH;
  static constexpr int OFF_ROW = OFF_EXP + M * 4;
  static constexpr int SMEM = OFF_ROW + M * 4;
};

template <int X>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (X == 2)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Two 16-bit numbers of type X in one word, and back.
template <int X>
__device__ __forceinline__ uint16_t bits16(float v) {
  if constexpr (X == 1) return __half_as_ushort(__float2half_rn(v));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
template <int X>
__device__ __forceinline__ float from16(uint16_t b) {
  if constexpr (X == 1) return __half2float(__ushort_as_half(b));
  else return __bfloat162float(__ushort_as_bfloat16(b));
}

// Two columns of y; aligned: one access of both.
template <int Y>
__device__ __forceinline__ float2 load2(const typename Val<Y>::type* p, bool aligned, bool second) {
  if (aligned && second) {
    if constexpr (Y == 0) return *reinterpret_cast<const float2*>(p);
    else {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
      return make_float2(from16<Y>(static_cast<uint16_t>(u)), from16<Y>(static_cast<uint16_t>(u >> 16)));
    }
  }
  return make_float2(Val<Y>::load(p), second ? Val<Y>::load(p + 1) : 0.0f);
}
template <int Y>
__device__ __forceinline__ void store2(typename Val<Y>::type* p, float2 v, bool aligned, bool second) {
  if (aligned && second) {
    if constexpr (Y == 0) *reinterpret_cast<float2*>(p) = v;
    else *reinterpret_cast<uint32_t*>(p) = bits16<Y>(v.x) | (static_cast<uint32_t>(bits16<Y>(v.y)) << 16);
    return;
  }
  *p = Val<Y>::to(v.x);
  if (second) p[1] = Val<Y>::to(v.y);
}

template <int X, int Y, int MT, int RP>
__global__ void __launch_bounds__(kThreads) lora_kernel(const LoraArgs p) {
  using Sh = LoraShape<MT, RP>;
  using YV = typename Val<Y>::type;
  constexpr int M = Sh::M, SPLIT = Sh::SPLIT, N8 = RP / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);
  float* sum = reinterpret_cast<float*>(smem + Sh::OFF_SUM);
  float* power = reinterpret_cast<float*>(smem + Sh::OFF_EXP);
  int* row_of = reinterpret_cast<int*>(smem + Sh::OFF_ROW);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3;
  const int rank = static_cast<int>(cluster_ctarank());
  const int rg = warp % MT, split = warp / MT;

  const GroupTile t = find_group_tile(p.offsets, p.groups, p.T, blockIdx.x / kRanks, M);
  if (t.group < 0) return;  // (all eight CTAs)
  const bool live = t.group < p.groups;
  if (!live && p.resid == p.y) return;
  for (int i = threadIdx.x; i < M; i += kThreads) {
    int r = -1;
    if (t.begin + i < t.end) {
      r = __ldg(p.order + t.begin + i);
      if (r < 0 || r >= p.T) r = -1;
    }
    row_of[i] = r;
  }
  __syncthreads();
  const int64_t n_slice = ((p.N + kRanks - 1) / kRanks + 31) / 32 * 32;
  const int64_t n0 = min(p.N, rank * n_slice), n1 = min(p.N, n0 + n_slice);
  const int row_a = row_of[rg * 16 + g], row_b = row_of[rg * 16 + g + 8];

  if (live) {
    // ------------------------------------------------------ 1: this CTA's eighth of K
    const int64_t k_slice = ((p.K + kRanks - 1) / kRanks + kStageK - 1) / kStageK * kStageK;
    const int64_t k0 = min(p.K, rank * k_slice), k1 = min(p.K, k0 + k_slice);
    const uint16_t* x = static_cast<const uint16_t*>(p.x);
    const uint16_t* a = static_cast<const uint16_t*>(p.a) + static_cast<int64_t>(t.group) * p.rank * p.K;
    float acc[N8][4] = {};
    if constexpr (MT == 1) {
      const uint16_t* xa = x + (row_a < 0 ? 0 : row_a) * p.ldx + q * 8;
      const uint16_t* xb = x + (row_b < 0 ? 0 : row_b) * p.ldx + q * 8;
#pragma unroll 2
      for (int64_t k = k0 + warp * 32; k < k1; k += kWarps * 32) {
        const bool in = k + q * 8 < k1;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 u = in && row_a >= 0 ? __ldg(reinterpret_cast<const uint4*>(xa + k)) : zero;
        const uint4 v = in && row_b >= 0 ? __ldg(reinterpret_cast<const uint4*>(xb + k)) : zero;
        uint4 w[N8];
#pragma unroll
        for (int j = 0; j < N8; ++j)
          w[j] = in && j * 8 < p.rank ? __ldg(reinterpret_cast<const uint4*>(a + (j * 8 + g) * p.K + k + q * 8)) : zero;
        const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
        for (int j = 0; j < N8; ++j) {
          mma16<X>(acc[j], a0, w[j].x, w[j].y);
          mma16<X>(acc[j], a1, w[j].z, w[j].w);
        }
      }
    } else {
      // x rows and A's rows, 64 of K a stage; odd rows have their halves swapped.
      constexpr int ROWS = M + RP, STAGE = ROWS * 128, PIECES = (ROWS * 8 + kThreads - 1) / kThreads;
      const uint32_t base = smem_u32(smem);
      const uint16_t* src[PIECES];
      bool there[PIECES];
      const int c = threadIdx.x & 7;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int r = (threadIdx.x >> 3) + i * (kThreads / 8);
        src[i] = x;
        there[i] = false;
        if (r < M) {
          there[i] = row_of[r] >= 0;
          if (there[i]) src[i] = x + row_of[r] * p.ldx;
        } else if (r < ROWS && r - M < p.rank) {
          there[i] = true;
          src[i] = a + static_cast<int64_t>(r - M) * p.K;
        }
      }
      int stage_in = 0;
      int64_t k_in = k0;
      auto ask = [&]() {
        if (k_in < k1) {
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            const int r = (threadIdx.x >> 3) + i * (kThreads / 8);
            if (r < ROWS) {
              const bool in = there[i] && k_in + c * 8 < k1;
              cp16(base + stage_in * STAGE + r * 128 + ((c ^ ((r & 1) << 2)) << 4), src[i] + (in ? k_in + c * 8 : 0), in);
            }
          }
          k_in += kStageK;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
      };
      for (int i = 0; i < kStages - 1; ++i) ask();
      int stage = 0;
      for (int64_t k = k0; k < k1; k += kStageK) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // the stage has arrived, and the one before it has been read
        ask();
        const uint8_t* sp = smem + stage * STAGE + (((split * 4 + q) ^ ((g & 1) << 2)) << 4);
        const uint4 u = *reinterpret_cast<const uint4*>(sp + (rg * 16 + g) * 128);
        const uint4 v = *reinterpret_cast<const uint4*>(sp + (rg * 16 + g + 8) * 128);
        const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
        for (int j = 0; j < N8; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(sp + (M + j * 8 + g) * 128);
          mma16<X>(acc[j], a0, w.x, w.y);
          mma16<X>(acc[j], a1, w.z, w.w);
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
      __syncthreads();  // the stages become the partial sums
    }
#pragma unroll
    for (int j = 0; j < N8; ++j) {
      float* d = part + (warp * 16 + g) * RP + j * 8 + 2 * q;
      *reinterpret_cast<float2*>(d) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(d + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < M * RP; i += kThreads) {
      const int m = i / RP, r = i % RP;
      float v = 0.0f;
#pragma unroll
      for (int s = 0; s < SPLIT; ++s) v += part[((s * MT + m / 16) * 16 + (m & 15)) * RP + r];
      sum[i] = v;
    }
    cluster_sync();
    // --------------------------- 2: this CTA's rows, from all eight and to all eight
    const float scale = p.scales ? __ldg(p.scales + t.group) : 1.0f;
    constexpr int MINE = M / kRanks, PER = RP >= 64 ? RP / 32 : 2, LANES = RP / PER;  // rows; values of a lane
    for (int i = warp; i < MINE; i += kWarps) {
      const int m = rank * MINE + i;
      float v[PER] = {};
      if (lane < LANES) {
#pragma unroll
        for (int s = 0; s < kRanks; ++s) {
          const uint32_t from = cluster_addr(sum + m * RP + lane * PER, s);
#pragma unroll
          for (int e = 0; e < PER; e += 2) {
            float2 w;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(w.x), "=f"(w.y) : "r"(from + e * 4) : "memory");
            v[e] += w.x;
            v[e + 1] += w.y;
          }
        }
      }
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        v[e] *= scale;
        top = fmaxf(top, fabsf(v[e]));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // 2^e >= top: the row's numbers are at most 1.  (fmaxf passes over NaN; a row with an infinity keeps its values.)
      int e2 = 0;
      if (top > 0.0f && top < INFINITY) frexpf(top, &e2);
      e2 = max(-126, min(126, e2));
      const float down = __int_as_float((127 - e2) << 23);
      uint32_t hi[PER / 2], lo[PER / 2];
#pragma unroll
      for (int e = 0; e < PER; e += 2) {
        uint16_t h[2], l[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const float w = v[e + i2] * down;
          h[i2] = bits16<X>(w);
          const float rest = w - from16<X>(h[i2]);
          l[i2] = bits16<X>(fabsf(w) < INFINITY ? rest : 0.0f);
        }
        hi[e / 2] = h[0] | (static_cast<uint32_t>(h[1]) << 16);
        lo[e / 2] = l[0] | (static_cast<uint32_t>(l[1]) << 16);
      }
      const float up = __int_as_float((127 + e2) << 23);
#pragma unroll
      for (int s = 0; s < kRanks; ++s) {
        if (lane < LANES) {
          const uint32_t to = cluster_addr(smem + Sh::OFF_H + m * Sh::PITCH + lane * PER * 2, s);
#pragma unroll
          for (int e = 0; e < PER / 2; ++e) {
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + e * 4), "r"(hi[e]) : "memory");
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + M * Sh::PITCH + e * 4), "r"(lo[e]) : "memory");
          }
        }
        if (lane == 0)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr(power + m, s)), "f"(up) : "memory");
      }
    }
    cluster_sync();
  }

  // -------------------------------------------- 3: this CTA's eighth of the columns
  const uint16_t* b = static_cast<const uint16_t*>(p.b) + static_cast<int64_t>(live ? t.group : 0) * p.N * p.rank;
  const uint8_t* h = smem + Sh::OFF_H + (rg * 16 + g) * Sh::PITCH;
  const float up_a = live ? power[rg * 16 + g] : 0.0f, up_b = live ? power[rg * 16 + g + 8] : 0.0f;
  constexpr int YS = static_cast<int>(sizeof(YV));
  const bool aligned = (reinterpret_cast<uintptr_t>(p.resid) | reinterpret_cast<uintptr_t>(p.y) |
                        static_cast<uintptr_t>(p.ldr * YS) | static_cast<uintptr_t>(p.ldy * YS)) % (2 * YS) == 0;
  if (rg * 16 >= t.end - t.begin) return;  // (nothing below waits)
  for (int64_t n = n0 + split * 32; n < n1; n += SPLIT * 32) {
    float2 ya[4], yb[4];
    float acc[4][4] = {};
    const YV* ra = static_cast<const YV*>(p.resid) + (row_a < 0 ? 0 : row_a) * p.ldr;
    const YV* rb = static_cast<const YV*>(p.resid) + (row_b < 0 ? 0 : row_b) * p.ldr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t col = n + j * 8 + 2 * q;
      ya[j] = yb[j] = make_float2(0.0f, 0.0f);
      if (col < n1 && row_a >= 0) ya[j] = load2<Y>(ra + col, aligned, col + 1 < n1);
      if (col < n1 && row_b >= 0) yb[j] = load2<Y>(rb + col, aligned, col + 1 < n1);
    }
    if (live) {
      if constexpr (RP == 16) {
        uint2 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t col = n + j * 8 + g;
          w[j] = col < n1 && q * 4 < p.rank ? __ldg(reinterpret_cast<const uint2*>(b + col * p.rank + q * 4)) : make_uint2(0, 0);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {  // the numbers, then what rounding them left
          const uint2 u = *reinterpret_cast<const uint2*>(h + s * M * Sh::PITCH + q * 8);
          const uint2 v = *reinterpret_cast<const uint2*>(h + s * M * Sh::PITCH + 8 * Sh::PITCH + q * 8);
          const uint32_t a0[4] = {u.x, v.x, u.y, v.y};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16<X>(acc[j], a0, w[j].x, w[j].y);
        }
      } else {
#pragma unroll
        for (int kb = 0; kb < RP / 32; ++kb) {
          uint4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int64_t col = n + j * 8 + g;
            w[j] = col < n1 && kb * 32 + q * 8 < p.rank
                       ? __ldg(reinterpret_cast<const uint4*>(b + col * p.rank + kb * 32 + q * 8)) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint4 u = *reinterpret_cast<const uint4*>(h + s * M * Sh::PITCH + kb * 64 + q * 16);
            const uint4 v = *reinterpret_cast<const uint4*>(h + s * M * Sh::PITCH + 8 * Sh::PITCH + kb * 64 + q * 16);
            const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma16<X>(acc[j], a0, w[j].x, w[j].y);
              mma16<X>(acc[j], a1, w[j].z, w[j].w);
            }
          }
        }
      }
    }
    YV* oa = static_cast<YV*>(p.y) + (row_a < 0 ? 0 : row_a) * p.ldy;
    YV* ob = static_cast<YV*>(p.y) + (row_b < 0 ? 0 : row_b) * p.ldy;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t col = n + j * 8 + 2 * q;
      if (col >= n1) continue;
      // (rows of no adapter stay as they are, to the bit)
      if (live) {
        ya[j] = make_float2(fmaf(up_a, acc[j][0], ya[j].x), fmaf(up_a, acc[j][1], ya[j].y));
        yb[j] = make_float2(fmaf(up_b, acc[j][2], yb[j].x), fmaf(up_b, acc[j][3], yb[j].y));
      }
      if (row_a >= 0) store2<Y>(oa + col, ya[j], aligned, col + 1 < n1);
      if (row_b >= 0) store2<Y>(ob + col, yb[j], aligned, col + 1 < n1);
    }
  }
}

template <int X, int Y, int MT, int RP>
cudaError_t launch_shape(const LoraArgs& a, cudaStream_t s) {
  using Sh = LoraShape<MT, RP>;
  static_assert(Sh::SMEM <= 227 * 1024, "shared memory");
  constexpr auto k = lora_kernel<X, Y, MT, RP>;
  if (cudaError_t e = allow_smem<k>(Sh::SMEM)) return e;
  const int64_t tiles = a.T / Sh::M + std::min<int64_t>(a.groups + 1, a.T);
  if (tiles > INT32_MAX / kRanks) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kRanks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * kRanks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Sh::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, a);
}

template <int X, int Y>
cudaError_t launch_types(const LoraArgs& a, cudaStream_t s) {
  // Tiles of 64 rows where the adapters have more than a few rows each, on average.
  if (a.T > 16 * a.groups) {
    if (a.rank <= 16) return launch_shape<X, Y, 4, 16>(a, s);
    if (a.rank <= 32) return launch_shape<X, Y, 4, 32>(a, s);
    if (a.rank <= 64) return launch_shape<X, Y, 4, 64>(a, s);
    return launch_shape<X, Y, 4, 128>(a, s);
  }
  if (a.rank <= 16) return launch_shape<X, Y, 1, 16>(a, s);
  if (a.rank <= 32) return launch_shape<X, Y, 1, 32>(a, s);
  if (a.rank <= 64) return launch_shape<X, Y, 1, 64>(a, s);
  return launch_shape<X, Y, 1, 128>(a, s);
}

}  // namespace

cudaError_t launch_lora(const LoraArgs& a, int xtype, int ytype, int num_sms, cudaStream_t s) {
  (void)num_sms;
  if (xtype == kXF16) return ytype == kXF32 ? launch_types<1, 0>(a, s) : launch_types<1, 1>(a, s);
  return ytype == kXF32 ? launch_types<2, 0>(a, s) : launch_types<2, 2>(a, s);
}

}  // namespace b2q
